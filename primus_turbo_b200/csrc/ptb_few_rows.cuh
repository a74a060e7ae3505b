// Products of a few rows of activations with a large weight, out[m, n] = sum_k x[m, k] * w[n, k], for weights of 16, 8 or 4 bits:
// what the 4-bit product and the MoE layer for few tokens share.
//
// Such a product reads the weight once and does little with it, so it is bound by HBM, and everything here serves to have
// many wide loads in flight.  The weight takes the 16-row side of mma.m16n8k16 and eight rows of x the other: tcgen05 wants 128
// weight rows and its operands in shared memory, which at one to eight rows buys nothing but a copy.  A warp walks 128-wide blocks
// of k; weights go from memory straight to the registers of the lane that feeds them to the MMA, 16 bytes at a time.
//
// The order of k inside an MMA is free as long as both operands agree on it.  Lane (g, t) = (lane / 4, lane % 4) of a warp
// supplies weight rows g and g + 8 and row g of x, four k per MMA.  An "octet" is the eight neighbouring k that a lane feeds to two
// MMAs; a block of 128 is four octets a lane.  Where octet q of lane t lies:
//   16-bit and 4-bit weights  k = 32 q + 8 t              (an MMA pair covers 32 neighbouring k: the smallest 4-bit group)
//   8-bit weights             k = 64 (q / 2) + 16 t + 8 (q % 2)   (16 bytes a lane and load)
// 4-bit weights are stored so that a lane's four octets are 16 neighbouring bytes (see Int4 below).
#pragma once

#include "ptb_common.cuh"

#include <type_traits>

namespace ptb {
namespace {

enum WeightFormat { kW16 = 0, kWE4M3 = 1, kWE5M2 = 2, kWInt4 = 3 };
constexpr int kKB = 128; // k per block

// 16 bytes that are read once: they pass by L1, where x stays
__device__ __forceinline__ uint4 load_once(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

template <typename T> __device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- 4-bit weights ------------------------------------------------------------------------------------------------
// Row n of a [N, K] weight is ceil(K / 128) blocks of 64 bytes.  The 16 octets of a block, octet (q, t) = k 32 q + 8 t ...,
// are 32-bit words; word t * 4 + q holds octet (q, t), so lane t of a quad reads its four octets as one 16-byte piece.  In a word
// the codes of k + 0 .. 7 sit in nibbles 0 4 1 5 2 6 3 7: masking with 0x000f000f after a shift by 0, 4, 8, 12 gives the pairs
// (k, k+1), (k+2, k+3) ... in the halves of a register, which is how the MMA takes them.  Codes past K are 0.
//   value = (code - zero) * scale, zero = 8 where no zero points are given.
constexpr int kInt4BlockBytes = 64;

// code pair -> (code - zero) in T's format, exactly: 128 + code is a bf16 with code in its low mantissa bits (1024 + code in fp16)
template <typename T> struct Int4Pair;
template <> struct Int4Pair<__nv_bfloat16> {
    static constexpr uint32_t kMagic = 0x43004300u;
    static __device__ __forceinline__ uint32_t sub(uint32_t v, uint32_t z) {
        uint32_t r;
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(z));
        return r;
    }
};
template <> struct Int4Pair<__half> {
    static constexpr uint32_t kMagic = 0x64006400u;
    static __device__ __forceinline__ uint32_t sub(uint32_t v, uint32_t z) {
        uint32_t r;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(z));
        return r;
    }
};

template <typename T> __device__ __forceinline__ uint32_t int4_zero(uint32_t z) { return Int4Pair<T>::kMagic | z | z << 16; }

template <typename T> __device__ __forceinline__ void int4_octet(uint32_t w, uint32_t zero, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = Int4Pair<T>::sub((w >> (4 * i) & 0x000f000fu) | Int4Pair<T>::kMagic, zero);
}

// ---- 8-bit weights --------------------------------------------------------------------------------------------------
// Four FP8 values -> two pairs of T.  Every e4m3 and e5m2 value, NaN and infinity too, is one of fp16; and of bf16, by way of fp32.
template <typename T, int FMT> __device__ __forceinline__ void fp8_pairs(uint32_t w, uint32_t &p0, uint32_t &p1) {
    uint32_t h0, h1;
    const uint16_t w0 = (uint16_t) w, w1 = (uint16_t) (w >> 16);
    if constexpr (FMT == kWE4M3) {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h0) : "h"(w0));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h1) : "h"(w1));
    } else {
        asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h0) : "h"(w0));
        asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h1) : "h"(w1));
    }
    if constexpr (std::is_same<T, __half>::value) {
        p0 = h0;
        p1 = h1;
    } else {
        const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&h0)), f1 = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
        const __nv_bfloat162 b0 = __float22bfloat162_rn(f0), b1 = __float22bfloat162_rn(f1);
        p0 = *reinterpret_cast<const uint32_t *>(&b0);
        p1 = *reinterpret_cast<const uint32_t *>(&b1);
    }
}

// ---- one weight row's share of a lane in a block ----------------------------------------------------------------------
template <int FMT> struct RowPiece {
    static constexpr int kVecs = FMT == kWInt4 ? 1 : FMT == kW16 ? 4 : 2;
    uint4 v[kVecs];
    // row: the row's first byte; K: the row's length (16-bit and 8-bit rows end at K, which is a multiple of 8 and 16)
    __device__ __forceinline__ void load(const uint8_t *row, int kb, int t, int K) {
        if constexpr (FMT == kWInt4) {
            v[0] = load_once(row + (int64_t) kb * kInt4BlockBytes + t * 16);
        } else if constexpr (FMT == kW16) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = kb * kKB + 32 * q + 8 * t;
                v[q] = k < K ? load_once(row + (int64_t) k * 2) : make_uint4(0, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int k = kb * kKB + 64 * q + 16 * t;
                v[q] = k < K ? load_once(row + k) : make_uint4(0, 0, 0, 0);
            }
        }
    }
    // octet q as four pairs of T
    template <typename T> __device__ __forceinline__ void octet(int q, uint32_t zero, uint32_t (&p)[4]) const {
        if constexpr (FMT == kWInt4) {
            const uint32_t w = q == 0 ? v[0].x : q == 1 ? v[0].y : q == 2 ? v[0].z : v[0].w;
            int4_octet<T>(w, zero, p);
        } else if constexpr (FMT == kW16) {
            p[0] = v[q].x; p[1] = v[q].y; p[2] = v[q].z; p[3] = v[q].w;
        } else {
            const uint4 u = v[q / 2];
            fp8_pairs<T, FMT>(q % 2 ? u.z : u.x, p[0], p[1]);
            fp8_pairs<T, FMT>(q % 2 ? u.w : u.y, p[2], p[3]);
        }
    }
};

template <int FMT> __device__ __forceinline__ int octet_k(int q, int t) { // where octet q of lane t starts in its block
    return FMT == kWE4M3 || FMT == kWE5M2 ? 64 * (q / 2) + 16 * t + 8 * (q % 2) : 32 * q + 8 * t;
}

// ---- scales -------------------------------------------------------------------------------------------------------------
// G: k per scale.  16-bit weights have none; 8-bit ones a float per block of 128 (whatever the granularity: a scale per row or
// tensor is found again at a stride of 0); 4-bit ones a bf16 per group and perhaps a zero point.
template <int FMT> struct RowScale {
    const float *s8;
    const __nv_bfloat16 *s4;
    const uint8_t *z4;
    int stride; // of s8, from block to block
    int count;  // of s4 and z4
    __device__ __forceinline__ float at(int group) const {
        if constexpr (FMT == kWInt4) return group < count ? __bfloat162float(s4[group]) : 0.0f;
        else return s8[(int64_t) group * stride];
    }
    __device__ __forceinline__ uint32_t zero(int group) const { return z4 != nullptr && group < count ? z4[group] : 8; }
};

// acc[i] += the product of one block of two weight rows a lane (pa, pb: rows g and g + 8 of the warp's 16) with NT * 8 rows of x.
// x(i, q, h) gives the lane's octet q of row g of the i-th eight, already in the block; kTerms of them (h) add up to x.
// Between two scales the MMA adds up products of x with the bare codes, which are exact in T; scaling is in 32 bits.
template <typename T, int FMT, int G, int NT, int kTerms, typename X>
__device__ __forceinline__ void few_rows_block(float (&acc)[NT][4], int kb, const RowPiece<FMT> &pa, const RowPiece<FMT> &pb,
                                               const RowScale<FMT> &sa, const RowScale<FMT> &sb, X &&x) {
    constexpr bool kScaled = FMT != kW16;
    constexpr int kPer = kScaled ? G / 32 : 4; // octets per scale
    float c[NT][4];
    uint32_t za = 0, zb = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int group = kb * (4 / kPer) + q / kPer;
        if (q % kPer == 0) {
            if constexpr (kScaled) {
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[i][j] = 0.0f;
            }
            if constexpr (FMT == kWInt4) {
                za = int4_zero<T>(sa.zero(group));
                zb = int4_zero<T>(sb.zero(group));
            }
        }
        uint32_t ua[4], ub[4];
        pa.template octet<T>(q, za, ua);
        pb.template octet<T>(q, zb, ub);
        const uint32_t f0[4] = {ua[0], ub[0], ua[1], ub[1]}, f1[4] = {ua[2], ub[2], ua[3], ub[3]};
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            float(&d)[4] = kScaled ? c[i] : acc[i];
#pragma unroll
            for (int h = 0; h < kTerms; ++h) {
                const uint4 u = x(i, q, h);
                mma_16816<T>(d, f0, u.x, u.y);
                mma_16816<T>(d, f1, u.z, u.w);
            }
        }
        if constexpr (kScaled) {
            if (q % kPer == kPer - 1) {
                const float ga = sa.at(group), gb = sb.at(group);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    acc[i][0] += c[i][0] * ga;
                    acc[i][1] += c[i][1] * ga;
                    acc[i][2] += c[i][2] * gb;
                    acc[i][3] += c[i][3] * gb;
                }
            }
        }
    }
}

} // namespace
} // namespace ptb
