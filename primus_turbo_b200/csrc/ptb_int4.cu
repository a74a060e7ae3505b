// 4-bit weights: quantise, dequantise, and the product of a few rows with one.  The layout is described in ptb_few_rows.cuh.
#include "ptb_few_rows.cuh"

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
            word |= (uint32_t) c << ((j / 2 + (j & 1) * 4) * 4);
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
    for (int j = 0; j < 8; ++j) r[j] = from_f32<T>((float) ((int) (word >> ((j / 2 + (j & 1) * 4) * 4) & 15) - z) * s);
    uint4 u[sizeof(T) / 2];
    memcpy(u, r, sizeof(r));
    uint4 *p = reinterpret_cast<uint4 *>(out + row * K + k);
#pragma unroll
    for (int j = 0; j < (int) sizeof(T) / 2; ++j) p[j] = u[j];
}

// ---- product of a few rows ----------------------------------------------------------------------------------------------
struct Int4GemmArgs {
    const void *x;
    int64_t ldx; // elements
    int M, N, K;
    const uint8_t *codes;
    const __nv_bfloat16 *scale;
    const uint8_t *zero;
    const void *bias;
    void *out;
};

constexpr int kGemmWarps = 8;

// One CTA: 16 weight rows against up to NT * 8 rows of x; its warps share the blocks of k and add up in shared memory in a fixed
// order.  Inside a group the codes less their zero are integers, so the MMA's sums are those of x times integers; each group's sum
// is scaled in 32 bits.
template <typename T, int G, int NT>
__global__ void __launch_bounds__(32 * kGemmWarps) int4_gemm_kernel(const Int4GemmArgs a) {
    grid_dep_begin();
    __shared__ float part[kGemmWarps][NT * 8][17];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (NT * 8);
    const int blocks = (a.K + kKB - 1) / kKB, groups = (a.K + G - 1) / G;
    const int ra = min(n0 + g, a.N - 1), rb = min(n0 + g + 8, a.N - 1);
    const uint8_t *wa = a.codes + (int64_t) ra * blocks * kInt4BlockBytes, *wb = a.codes + (int64_t) rb * blocks * kInt4BlockBytes;
    RowScale<kWInt4> sa{}, sb{};
    sa.s4 = a.scale + (int64_t) ra * groups;
    sb.s4 = a.scale + (int64_t) rb * groups;
    sa.count = sb.count = groups;
    if (a.zero != nullptr) {
        sa.z4 = a.zero + (int64_t) ra * groups;
        sb.z4 = a.zero + (int64_t) rb * groups;
    }
    const T *x[NT];
    bool live[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int m = m0 + i * 8 + g;
        live[i]     = m < a.M;
        x[i]        = (const T *) a.x + (live[i] ? m : 0) * a.ldx + 8 * t;
    }
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    auto block = [&](int kb, const RowPiece<kWInt4> &pa, const RowPiece<kWInt4> &pb) {
        few_rows_block<T, kWInt4, G, NT, 1>(acc, kb, pa, pb, sa, sb, [&](int i, int q, int) {
            const int k = kb * kKB + 32 * q;
            return live[i] && k + 8 * t < a.K ? *reinterpret_cast<const uint4 *>(x[i] + k) : make_uint4(0, 0, 0, 0);
        });
    };
    constexpr int kAhead = 4; // blocks whose weights are in flight
    for (int kb = warp; kb < blocks; kb += kGemmWarps * kAhead) {
        RowPiece<kWInt4> pa[kAhead], pb[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (kb + u * kGemmWarps < blocks) {
                pa[u].load(wa, kb + u * kGemmWarps, t, a.K);
                pb[u].load(wb, kb + u * kGemmWarps, t, a.K);
            }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (kb + u * kGemmWarps < blocks) block(kb + u * kGemmWarps, pa[u], pb[u]);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        part[warp][i * 8 + 2 * t][g]         = acc[i][0];
        part[warp][i * 8 + 2 * t + 1][g]     = acc[i][1];
        part[warp][i * 8 + 2 * t][g + 8]     = acc[i][2];
        part[warp][i * 8 + 2 * t + 1][g + 8] = acc[i][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 8 * 16; i += 32 * kGemmWarps) {
        const int m = i / 16, n = i % 16;
        if (m0 + m >= a.M || n0 + n >= a.N) continue;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kGemmWarps; ++w) s += part[w][m][n];
        if (a.bias != nullptr) s += to_f32(((const T *) a.bias)[n0 + n]);
        ((T *) a.out)[(int64_t) (m0 + m) * a.N + n0 + n] = from_f32<T>(s);
    }
}

template <typename T, int G> cudaError_t launch_gemm(const Int4GemmArgs &a, cudaStream_t st) {
    const unsigned gx = (unsigned) cdiv(a.N, 16);
    if (a.M <= 8) return launch_after(int4_gemm_kernel<T, G, 1>, dim3(gx, 1), 32 * kGemmWarps, 0, st, 1, a);
    if (a.M <= 16) return launch_after(int4_gemm_kernel<T, G, 2>, dim3(gx, 1), 32 * kGemmWarps, 0, st, 1, a);
    return launch_after(int4_gemm_kernel<T, G, 4>, dim3(gx, (unsigned) cdiv(a.M, 32)), 32 * kGemmWarps, 0, st, 1, a);
}

bool is_group(int64_t g) { return g == 32 || g == 64 || g == 128; }

#define PTB_SWITCH_INT4_GROUP(g, G, ...)                   \
    switch (g) {                                           \
    case 32: { constexpr int G = 32; __VA_ARGS__; } break; \
    case 64: { constexpr int G = 64; __VA_ARGS__; } break; \
    default: { constexpr int G = 128; __VA_ARGS__; }       \
    }

} // namespace
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

int ptb_gemm_int4(const void *x, int dtype, int64_t ldx, int64_t M, int64_t N, int64_t K, const void *codes, const void *scale, const void *zero,
                  int64_t group, const void *bias, void *out, ptb_stream_t stream) {
    PTB_REQUIRE(M >= 0 && N >= 0 && K >= 1, PTB_ERR_ARG, "gemm_int4: bad shape");
    PTB_REQUIRE(dtype == PTB_BF16 || dtype == PTB_F16, PTB_ERR_ARG, "gemm_int4: x must be bf16 or fp16");
    PTB_REQUIRE(is_group(group), PTB_ERR_ARG, "gemm_int4: the group size must be 32, 64 or 128");
    PTB_REQUIRE(K % 8 == 0 && (M <= 1 || ldx % 8 == 0), PTB_ERR_ALIGN, "gemm_int4: the row length and pitch of x must be multiples of 8");
    PTB_REQUIRE(M <= 1 || ldx >= K, PTB_ERR_ARG, "gemm_int4: rows of x overlap");
    PTB_REQUIRE(K <= 1 << 24 && N <= 1 << 30 && M <= 1 << 20, PTB_ERR_TOO_LARGE, "gemm_int4: matrix too large");
    if (M == 0 || N == 0) return 0;
    PTB_REQUIRE(x && codes && scale && out, PTB_ERR_ARG, "gemm_int4: null pointer");
    PTB_REQUIRE(aligned16(x) && aligned16(codes), PTB_ERR_ALIGN, "gemm_int4: x and the codes must be 16-byte aligned");
    const Int4GemmArgs a{x, ldx, (int) M, (int) N, (int) K, (const uint8_t *) codes, (const __nv_bfloat16 *) scale, (const uint8_t *) zero, bias, out};
    PTB_SWITCH_INT4_GROUP(group, G, {
        if (dtype == PTB_BF16) PTB_CUDA((launch_gemm<__nv_bfloat16, G>(a, (cudaStream_t) stream)));
        else PTB_CUDA((launch_gemm<__half, G>(a, (cudaStream_t) stream)));
    });
    PTB_LAUNCH_CHECK("int4_gemm_kernel");
    return 0;
}

#pragma GCC visibility pop
} // extern "C"
