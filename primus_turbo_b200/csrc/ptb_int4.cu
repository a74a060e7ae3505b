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
// One thread takes an octet (16 bytes of a 16-bit weight) and writes its 32-bit word; G / 8 neighbouring lanes share a group.
// HBM-bound: 2 bytes in and half a byte out for a value.

// rint(w / s) with the quotient correct to the last bit where it matters: next to a half-integer the sign of the exact remainder decides
__device__ __forceinline__ float code_steps(float w, float s, float inv) {
    float r       = rintf(w * inv);
    r             = fminf(fmaxf(r, -16.0f), 16.0f);
    const float d = __fmaf_rn(-r, s, w);   // w - r s, rounded once
    const float h = 0.5f * s;
    // |d| == s / 2 is the tie (to even); beyond it the product with the inverse was a rounding off
    if (fabsf(d) > h) r += d > 0.0f ? 1.0f : -1.0f;
    else if (fabsf(d) == h && (((int) r) & 1)) r += d > 0.0f ? 1.0f : -1.0f;
    return r;
}

template <typename T, int G, bool kZeros>
__global__ void __launch_bounds__(256) int4_quant_kernel(const T *w, int64_t octets_per_row, int64_t total, int K, uint32_t *codes,
                                                          __nv_bfloat16 *scale, uint8_t *zero) {
    grid_dep_begin();
    // thread -> octet of a padded row (a multiple of 16 octets): the lanes of a group are neighbours in a warp
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    const bool here = i < total;
    const int64_t row = here ? i / octets_per_row : 0;
    const int o = here ? (int) (i - row * octets_per_row) : 0;
    const int k = o * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (here && k < K) {
        const T *p = w + row * K + k;
        if constexpr (sizeof(T) == 2) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = to_f32(reinterpret_cast<const T *>(&u)[j]);
        } else {
            const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
    }
    float lo = 0.0f, hi = 0.0f; // of min(w, 0) and max(w, 0)
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, v[j]);
        hi = fmaxf(hi, v[j]);
        finite = finite && fabsf(v[j]) < INFINITY;
    }
    if (!finite) hi = INFINITY;
#pragma unroll
    for (int m = 1; m < G / 8; m <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
    const float wide = kZeros ? __fsub_rn(__fdiv_rn(hi, 15.0f), __fdiv_rn(lo, 15.0f)) : __fdiv_rn(fmaxf(hi, -lo), 7.0f);
    const bool fine  = hi < INFINITY;
    const __nv_bfloat16 sb = fine ? __float2bfloat16_rn(wide) : __float2bfloat16_rn(NAN);
    const float s = __bfloat162float(sb);
    int z = 8;
    if (kZeros) z = fine && s > 0.0f ? (int) fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.0f), 15.0f) : 0;
    uint32_t word = 0;
    if (fine && s > 0.0f) {
        const float inv = __fdiv_rn(1.0f, s);
        const bool plain = inv < INFINITY; // the inverse of a subnormal scale may overflow
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float steps = plain ? code_steps(v[j], s, inv) : rintf(fminf(fmaxf(__fdiv_rn(v[j], s), -16.0f), 16.0f));
            const int c       = min(max((int) steps + z, 0), 15);
            word |= (uint32_t) c << int4_shift(j);
        }
    } else {
        word = 0x11111111u * (uint32_t) z;
    }
    if (!here) return;
    if (k >= K) word = 0;
    // octet (q, t) of block b is word t * 4 + q
    const int64_t b = row * (octets_per_row / 16) + o / 16;
    codes[b * 16 + (o & 3) * 4 + ((o >> 2) & 3)] = word;
    const int groups = (K + G - 1) / G, g = k / G;
    if (o % (G / 8) == 0 && g < groups) {
        scale[row * groups + g] = sb;
        if (kZeros) zero[row * groups + g] = (uint8_t) z;
    }
}

// ---- dequantise --------------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) int4_dequant_kernel(const uint32_t *codes, const __nv_bfloat16 *scale, const uint8_t *zero, int G,
                                                            int64_t octets_per_row, int64_t total, int K, T *out) {
    grid_dep_begin();
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t row = i / octets_per_row;
    const int o = (int) (i - row * octets_per_row), k = o * 8;
    if (k >= K) return;
    const int groups = (K + G - 1) / G;
    const int64_t at = row * groups + k / G;
    const float s = __bfloat162float(scale[at]);
    const int z   = zero != nullptr ? zero[at] : 8;
    const uint32_t word = codes[(row * (octets_per_row / 16) + o / 16) * 16 + (o & 3) * 4 + ((o >> 2) & 3)];
    T r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = from_f32<T>((float) ((int) (word >> int4_shift(j) & 15) - z) * s);
    uint4 u[sizeof(T) / 2];
    memcpy(u, r, sizeof(r));
    uint4 *p = reinterpret_cast<uint4 *>(out + row * K + k);
#pragma unroll
    for (int j = 0; j < (int) sizeof(T) / 2; ++j) p[j] = u[j];
}

// ---- product of a few rows ----------------------------------------------------------------------------------------------
struct Int4GemmArgs {
    const void *x;
    int64_t ldx;
    ScaledRows xs;
    int M, N, K;
    const uint8_t *codes;
    const __nv_bfloat16 *scale;
    const uint8_t *zero;
    const void *bias;
    void *out;
};

template <int G> struct Int4Rows { // a lane's two rows of the weight
    const uint8_t *row[2];
    RowScale<kWInt4> scale[2];
    __device__ __forceinline__ void aim(const Int4GemmArgs &a, int n0) {
        const int blocks = (a.K + kKB - 1) / kKB, groups = (a.K + G - 1) / G;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t r = min(n0 + (((int) threadIdx.x & 31) >> 2) + 8 * h, a.N - 1);
            row[h]   = a.codes + r * blocks * kInt4BlockBytes;
            scale[h] = {nullptr, (const uint16_t *) a.scale + r * groups, a.zero ? a.zero + r * groups : nullptr, 0, groups};
        }
    }
};

// Up to eight rows, as far as they fit into shared memory.
template <int G> struct Int4TokenRows {
    const Int4GemmArgs &a;
    const uint8_t *row;
    RowScale<kWInt4> scale[2];
    __device__ __forceinline__ Int4TokenRows(const Int4GemmArgs &a) : a(a) {}
    __device__ __forceinline__ void open(int tile, int) {
        const int lane = threadIdx.x & 31, blocks = (a.K + kKB - 1) / kKB, groups = (a.K + G - 1) / G;
        row = a.codes + (int64_t) min(tile * 16 + (lane & 15), a.N - 1) * blocks * kInt4BlockBytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t r = min(tile * 16 + (lane >> 2) + 8 * h, a.N - 1);
            scale[h] = {nullptr, (const uint16_t *) a.scale + r * groups, a.zero ? a.zero + r * groups : nullptr, 0, groups};
        }
    }
};
template <typename T, int G> __global__ void __launch_bounds__(32 * kTokenWarps, 1) int4_token_kernel(const __grid_constant__ Int4GemmArgs a, int shares) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, blocks = (a.K + kKB - 1) / kKB;
    few_tokens_walk<T, kWInt4, G, 2, false, false, false>(
        smem, a.M, (a.N + 15) / 16, shares, 1, a.K, Int4TokenRows<G>(a),
        [&](uint8_t *x, uint8_t *runs) {
            stage_blocks<T, T, kWInt4, G, 2>(x, runs, blocks, a.M, [&](int block, int col, int &left) {
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

// More rows: a CTA has WR * 16 weight rows and up to NT * 8 rows of x; WK shares of k are added up in shared memory in a fixed order.
template <int G> struct Int4BatchRows : Int4Rows<G> {
    ScaledRows xs;
    int row0;
    __device__ __forceinline__ const uint8_t *x(int, int col) const { return xs.planes + (row0 + col) * xs.pitch; }
    __device__ __forceinline__ const float *runs(int col) const { return xs.runs + (int64_t) (row0 + col) * xs.blocks; }
};
template <typename T, int G, int NT, int WR, int WK, int kStages>
__global__ void __launch_bounds__(32 * WR * WK, 2) int4_gemm_kernel(const Int4GemmArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    using W = Walk<kWInt4, 128, WR, WK>;
    const int n0 = blockIdx.x * W::kRows, m0 = blockIdx.y * (NT * 8), cols = min(NT * 8, a.M - m0);
    Int4BatchRows<G> src;
    src.aim(a, n0 + (threadIdx.x >> 5) % WR * 16);
    src.xs   = a.xs;
    src.row0 = m0;
    float acc[NT][4] = {};
    few_rows_walk<T, kWInt4, G, 128, NT, WR, WK, kStages, 1, false>(acc, smem, a.K, cols, (cols + 7) / 8, src);
    const ShareSums<NT, WR, WK> sums(acc, smem);
    for (int i = threadIdx.x; i < cols * W::kRows; i += W::kThreads) {
        const int m = i / W::kRows, n = i % W::kRows;
        if (n0 + n >= a.N) continue;
        float s = sums.sum(m, n);
        if (a.bias != nullptr) s += to_f32(((const T *) a.bias)[n0 + n]);
        ((T *) a.out)[(int64_t) (m0 + m) * a.N + n0 + n] = from_f32<T>(s);
    }
}

template <typename T, int G, int NT, int WR, int WK, int kStages> cudaError_t launch_tile(const Int4GemmArgs &a, cudaStream_t st) {
    using W = Walk<kWInt4, 128, WR, WK>;
    const int smem = W::template smem<NT>(kStages, 1, (int) imin(a.M, NT * 8));
    return launch_early(int4_gemm_kernel<T, G, NT, WR, WK, kStages>, dim3((unsigned) cdiv(a.N, W::kRows), (unsigned) cdiv(a.M, NT * 8)), W::kThreads,
                        (size_t) smem, st, a);
}

constexpr int kMostSmem = 227 * 1024 - 1024; // of a CTA, less what is not dynamic

template <typename T, int G> int launch_gemm(const Int4GemmArgs &a, cudaStream_t st) {
    const int x_bytes = a.M <= kTokenCols && a.K <= 1 << 20 ? TokenX<kWInt4, G>::bytes(2, a.M, cdiv(a.K, kKB)) : kMostSmem;
    if (token_smem(x_bytes, a.M) <= kMostSmem) {
        int sms = 0;
        if (int rc = sm_count(&sms)) return rc;
        const int tiles = cdiv(a.N, 16), shares = token_shares(tiles, cdiv(a.K, kKB), sms);
        PTB_CUDA(launch_early(int4_token_kernel<T, G>, dim3((unsigned) cdiv(tiles, kTokenWarps >> shares)), 32 * kTokenWarps, (size_t) token_smem(x_bytes, a.M), st, a, shares));
        PTB_LAUNCH_CHECK("int4_token_kernel");
        return 0;
    }
    const int64_t warps = a.M * cdiv<int64_t>(a.K, kKB);
    PTB_CUDA(launch_early(scale_rows_kernel<T, kWInt4>, dim3((unsigned) cdiv<int64_t>(warps, 4)), 128, 0, st, (const T *) a.x, a.ldx, a.M, a.K, a.xs));
    PTB_LAUNCH_CHECK("scale_rows_kernel");
    if (a.M <= 8) PTB_CUDA((launch_tile<T, G, 1, 2, 4, 4>(a, st)));
    else if (a.M <= 16) PTB_CUDA((launch_tile<T, G, 2, 4, 2, 4>(a, st)));
    else PTB_CUDA((launch_tile<T, G, 4, 4, 2, 4>(a, st)));
    PTB_LAUNCH_CHECK("int4_gemm_kernel");
    return 0;
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
    const int64_t octets = cdiv<int64_t>(K, kKB) * 16, total = rows * octets;
    PTB_REQUIRE(total <= 256ll * 2147483647ll, PTB_ERR_TOO_LARGE, "quant_int4: too many values");
    const dim3 grid((unsigned) cdiv<int64_t>(total, 256));
    PTB_SWITCH_HP(dtype, T, PTB_SWITCH_INT4_GROUP(group, G, {
        if (zero != nullptr)
            PTB_CUDA(launch_after(int4_quant_kernel<T, G, true>, grid, 256, 0, (cudaStream_t) stream, 1, (const T *) w, octets, total, (int) K,
                                  (uint32_t *) codes, (__nv_bfloat16 *) scale, (uint8_t *) zero));
        else
            PTB_CUDA(launch_after(int4_quant_kernel<T, G, false>, grid, 256, 0, (cudaStream_t) stream, 1, (const T *) w, octets, total, (int) K,
                                  (uint32_t *) codes, (__nv_bfloat16 *) scale, (uint8_t *) nullptr));
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
    const int64_t octets = cdiv<int64_t>(K, kKB) * 16, total = rows * octets;
    PTB_REQUIRE(total <= 256ll * 2147483647ll, PTB_ERR_TOO_LARGE, "dequant_int4: too many values");
    const dim3 grid((unsigned) cdiv<int64_t>(total, 256));
    PTB_SWITCH_HP(out_dtype, T, PTB_CUDA(launch_after(int4_dequant_kernel<T>, grid, 256, 0, (cudaStream_t) stream, 1, (const uint32_t *) codes,
                                                       (const __nv_bfloat16 *) scale, (const uint8_t *) zero, (int) group, octets, total, (int) K, (T *) out)));
    PTB_LAUNCH_CHECK("int4_dequant_kernel");
    return 0;
}

int64_t ptb_gemm_int4_workspace(int dtype, int64_t M, int64_t K, int64_t group) {
    if (M < 0 || K < 1 || (dtype != PTB_BF16 && dtype != PTB_F16) || !is_group(group)) return -1;
    return scaled_bytes(1, M, K, 128);
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
    const Int4GemmArgs a{x, ldx, scaled_rows_at(workspace, 1, M, K), (int) M, (int) N, (int) K, (const uint8_t *) codes,
                         (const __nv_bfloat16 *) scale, (const uint8_t *) zero, bias, out};
    cudaStream_t st = (cudaStream_t) stream;
    PTB_SWITCH_INT4_GROUP(group, G, return dtype == PTB_BF16 ? launch_gemm<__nv_bfloat16, G>(a, st) : launch_gemm<__half, G>(a, st));
    return 0;
}

#pragma GCC visibility pop
} // extern "C"
