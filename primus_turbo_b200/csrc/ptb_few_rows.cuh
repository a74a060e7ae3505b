// Products of a few rows of activations with a large weight, out[m, n] = sum_k x[m, k] * w[n, k], for weights of 16, 8 or 4 bits:
// what the 4-bit product and the MoE layer for few tokens share.
//
// Such a product reads the weight once and does little with it, so it is bound by HBM, and everything here serves to have
// many wide loads in flight and few instructions per weight.  The weight takes the 16-row side of mma.sync and eight rows of x the
// other: tcgen05 wants 128 weight rows and its operands in shared memory, which at one to sixteen rows buys nothing but a copy.  A warp
// walks 128-wide blocks of k.  Weights travel by cp.async into shared-memory slots that belong to the lane that will feed them to the
// MMA, several blocks ahead, without holding registers and without a barrier: a lane reads back what it copied itself.
//
// What an MMA is fed with.  Measured on a B200, an SM issues an m16n8k16 of 16-bit floats or an m16n8k32 of bytes every 2.1 clocks (FP8
// ones are taken apart into these: 5.6), and integer and conversion instructions at 64 lanes a clock; HBM brings 23 bytes a clock
// and SM.  Unpacking 4-bit codes to bf16 is 7 such instructions for 8 codes, FP8 to bf16 8 for 4 values: too near the budget or beyond it.  So
//   * for a token or a few (few_tokens_walk) 4-bit codes go in as the bytes they are: two ANDs and a shift for 8 codes.  x is a 16-bit
//     integer per value, scaled by a power of two per block that brings the largest of its 128 to 2^14 .. 2^15, as a signed high byte
//     and an unsigned low one.  bf16's eight bits are exact in it down to 2^-7 of the largest; below, a value is off by up to 2^-15 of
//     the largest.  Sums of a group are exact integers, and scaling them is what costs: with more columns of x than eight it is too much;
//   * for more (few_rows_walk) codes become fp16 less their zero, exactly, 9 instructions for 8;
//   * FP8 weights are converted to fp16, exactly, one instruction for two;
//   * x goes with fp16 weights as fp16, scaled by a power of two per block into its range, where bf16 and fp16 values are exact down
//     to 2^-27 of the block's largest;
//   * 16-bit weights go in with 16-bit x as they are.
//
// The order of k inside an MMA is free as long as both operands agree on it.  Lane (g, t) = (lane / 4, lane % 4) of a warp supplies weight
// rows g and g + 8 and row g of x.  An "octet" is eight neighbouring k of a lane: one MMA of bytes, or two of 16 bits.  A block of
// 128 is four octets a lane.  Where octet q of lane t lies:
//   16-bit and 4-bit weights  k = 32 q + 8 t                    (octet q of all four lanes: 32 neighbouring k, the smallest 4-bit group)
//   8-bit weights             k = 64 (q / 2) + 16 t + 8 (q % 2) (16 bytes a lane and load; octets 2 c and 2 c + 1: 64 neighbouring k)
#pragma once

#include "ptb_common.cuh"

#include <type_traits>

namespace ptb {
namespace {

enum WeightFormat { kW16 = 0, kWE4M3 = 1, kWE5M2 = 2, kWInt4 = 3 };
constexpr int kKB = 128; // k per block
template <int FMT> constexpr bool kScaledX = FMT != kW16; // x is scaled per block

// 4-bit weights.  Row n of a [N, K] weight is ceil(K / 128) blocks of 64 bytes.  Word t * 4 + q of a block holds octet (q, t), so lane t
// of a quad reads its four octets as one 16-byte piece.  Byte i of a word holds code i of the eight in its low nibble and code
// i + 4 in its high one.  Codes past K are 0.   value = (code - zero) * scale, zero = 8 where no zero points are given.
constexpr int kInt4BlockBytes = 64;
__device__ __forceinline__ int int4_shift(int i) { return (i & 3) * 8 + (i >> 2) * 4; } // of code i of a word

// ---- launches that start under the kernel before ----------------------------------------------------------------------
// A kernel that is launched with launch_early may start once every CTA of the kernel before has called grid_dep_open.  That one calls it
// after its own grid_dep_wait: so when a CTA of this kernel runs, everything before the kernel before is done, and what does not come
// from that kernel -- the weights -- may be fetched ahead of grid_dep_wait.  Every CTA calls grid_dep_wait before it leaves.
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dep_open() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
inline cudaError_t launch_early(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, A &&...args) {
    if (smem > 32 * 1024) // 48 KB without asking, with what the kernel has besides
        if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem)) return e;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

inline int sm_count(int *sms) {
    int dev = 0;
    PTB_CUDA(cudaGetDevice(&dev));
    PTB_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    return 0;
}

// ---- copies -------------------------------------------------------------------------------------------------------------
// 16 bytes to shared memory past L1; zeros where nothing is there (nothing is read then)
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there = true) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); } // closes a batch
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t shared_u32(const void *p) { return (uint32_t) __cvta_generic_to_shared(p); }
__device__ __forceinline__ uint4 read16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float read4(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t read4u(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 read8u(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}

// ---- bulk copies and the barriers they complete on ---------------------------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_init_fence() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// 16-byte aligned addresses, a multiple of 16 bytes
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Gives up after two seconds; then the result is incomplete, and the status word (ptb_gemm_status) says so.
__device__ int g_few_status = 0;
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
    if (bar_try(bar, parity)) return true;
    uint64_t t0, now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 256; ++i)
            if (bar_try(bar, parity)) return true;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
        if (now - t0 > 2000000000ull) return false;
    }
}
// This file's status word: added to *status, cleared if asked for.
inline int few_status(int *status, int reset) {
    int code = 0;
    PTB_CUDA(cudaMemcpyFromSymbol(&code, g_few_status, sizeof(int)));
    if (code != 0) {
        *status        = code;
        const int zero = 0;
        if (reset) PTB_CUDA(cudaMemcpyToSymbol(g_few_status, &zero, sizeof(int)));
    }
    return 0;
}

// ---- MMAs: c += a * b ---------------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void mma_16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool kSigned> __device__ __forceinline__ void mma_8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (kSigned)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Sums of bytes start at this: an integer of up to 22 bits added to it is, read as a float, 1.5 * 2^23 plus that integer.
constexpr int kFloatBase = 0x4b400000;
constexpr float kFloatBaseValue = 12582912.0f;

// ---- scaled x -----------------------------------------------------------------------------------------------------------------
// scale and its inverse from the largest magnitude (finite): powers of two that bring it to [2^top, 2^(top + 1))
__device__ __forceinline__ void block_scale(float largest, int top, float &scale, float &inv) {
    const int e = max((int) (__float_as_uint(largest) >> 23), top + 1); // (values below 2^(top - 126) are left to their own)
    scale = __uint_as_float((uint32_t) (e - top) << 23);
    inv   = __uint_as_float((uint32_t) (254 + top - e) << 23);
}
constexpr int kTopInt = 14, kTopHalf = 13;
__device__ __forceinline__ int fixed16(float v) { return max(min(__float2int_rn(v), 32767), -32768); }
// Where value k of a block stands: among the bytes that go with byte codes (lane t's four octets are 32 neighbouring bytes), and among the
// fp16 that go with 4-bit weights (an octet in the order 0 2 1 3 4 6 5 7) or 8-bit ones (in the order of k).
__host__ __device__ __forceinline__ int byte_place(int k) { return (k / 8 % 4) * 32 + (k / 32) * 8 + k % 8; }
template <int FMT> __host__ __device__ __forceinline__ int half_place(int k) { return FMT == kWInt4 ? (k & ~3) | (k & 1) << 1 | (k & 2) >> 1 : k; }

// ---- one weight row's share of a lane in a block ----------------------------------------------------------------------
template <int FMT> struct RowPiece {
    static constexpr int kVecs = FMT == kWInt4 ? 1 : FMT == kW16 ? 4 : 2;
    uint4 v[kVecs];
    static constexpr int kBlockBytes = FMT == kWInt4 ? kInt4BlockBytes : FMT == kW16 ? 256 : 128;
    // at: the lane's first 16 bytes of the block; slot: where they go, the next ones 512 bytes on
    static __device__ __forceinline__ void copy(uint32_t slot, const uint8_t *at) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) copy16(slot + i * 512, at + i * 64);
    }
    // the same of a row's last block, where 16-bit and 8-bit rows end after `left` values
    static __device__ __forceinline__ void copy_last(uint32_t slot, const uint8_t *at, int t, int left) {
        constexpr int kStep = FMT == kW16 ? 32 : 64; // values from piece to piece
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const bool there = i * kStep + t * (kStep / 4) < left;
            copy16(slot + i * 512, there ? at + i * 64 : at, there);
        }
    }
    __device__ __forceinline__ void read(uint32_t slot) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i] = read16(slot + i * 512);
    }
    // from rows as they are: `at` is the lane's first 16 bytes, the next ones 64 on
    __device__ __forceinline__ void read_row(uint32_t at) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i] = read16(at + i * 64);
    }
    // zeros past the first `left` values of a block
    __device__ __forceinline__ void cut(int t, int left) {
        constexpr int kStep = FMT == kW16 ? 32 : 64;
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
            if (i * kStep + t * (kStep / 4) >= left) v[i] = make_uint4(0, 0, 0, 0);
    }
    // 4-bit: the eight bytes of octet q
    __device__ __forceinline__ void bytes(int q, uint32_t &lo, uint32_t &hi) const {
        const uint32_t w = q == 0 ? v[0].x : q == 1 ? v[0].y : q == 2 ? v[0].z : v[0].w;
        lo = w & 0x0f0f0f0fu;
        hi = w >> 4 & 0x0f0f0f0fu;
    }
    // octet q as four pairs of fp16.  4-bit: code - zero, in the order 0 2, 1 3, 4 6, 5 7.  A code in the low bits of 1024's mantissa is
    // 1024 + code, four bits higher 1024 + 16 code: one fma takes the base off either.  za, zb: -(1024 + zero) and -(64 + zero) in both halves.
    __device__ __forceinline__ void halves(int q, uint32_t za, uint32_t zb, uint32_t (&p)[4]) const {
        if constexpr (FMT == kWInt4) {
            const uint32_t w = q == 0 ? v[0].x : q == 1 ? v[0].y : q == 2 ? v[0].z : v[0].w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = ((i & 1 ? w >> 8 : w) & (i < 2 ? 0x000f000fu : 0x00f000f0u)) | 0x64006400u;
                asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(p[i]) : "r"(u), "r"(i < 2 ? 0x3c003c00u : 0x2c002c00u), "r"(i < 2 ? za : zb)); // times 1 or 1 / 16
            }
        } else {
            const uint4 u = v[q / 2 % kVecs];
            const uint32_t w[2] = {q % 2 ? u.z : u.x, q % 2 ? u.w : u.y};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t b = (uint16_t) (w[i / 2] >> (16 * (i % 2)));
                if constexpr (FMT == kWE5M2) asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(p[i]) : "h"(b));
                else asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p[i]) : "h"(b));
            }
        }
    }
};
// -(base + zero) in both halves, base 1024 or 64: fp16 numbers whose last bit is worth 1 or 1 / 16
__device__ __forceinline__ uint32_t minus_zero(uint32_t z, int base) { return (base == 1024 ? 0xe400u + z : 0xd400u + 16 * z) * 0x00010001u; }

// ---- scales of a weight ---------------------------------------------------------------------------------------------------
// 16-bit weights have none; 8-bit ones a float per block of 128 (whatever the granularity: a scale per row or tensor is found again
// at a stride of 0); 4-bit ones a bf16 and perhaps a zero point per group of G.
template <int FMT> struct RowScale { // one row's
    const float *s8;
    const uint16_t *s4;
    const uint8_t *z4;
    int stride; // of s8, from block to block
    int count;  // of s4 and z4
};
// One block's, in registers: asked for a block ahead, as they are stored; what is made of them waits until they are there.
template <int FMT, int G> struct BlockScale {
    static constexpr int kN = FMT == kWInt4 ? kKB / G : 1;
    uint16_t s4[kN];
    uint8_t z4[kN];
    float s8;
    // r: the row's scales from block kb on; `last`: there may be fewer than a block's (past the last group x is zero)
    __device__ __forceinline__ void load(const RowScale<FMT> &r, int kb, bool last) {
        if constexpr (FMT == kWInt4) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int g = kN > 1 && last ? min(i, r.count - 1 - kb * kN) : i;
                s4[i] = r.s4[g];
                z4[i] = 8;
                if (r.z4 != nullptr) z4[i] = r.z4[g];
            }
        } else if constexpr (FMT != kW16) {
            s8 = *r.s8;
        }
    }
    static __device__ __forceinline__ void advance(RowScale<FMT> &r, int blocks) {
        if constexpr (FMT == kWInt4) {
            r.s4 += blocks * kN;
            if (r.z4 != nullptr) r.z4 += blocks * kN;
        } else if constexpr (FMT != kW16) {
            r.s8 += blocks * r.stride;
        }
    }
    __device__ __forceinline__ float zero(int i) const { return (float) z4[i]; }
    __device__ __forceinline__ float scale(int i) const { return FMT == kWInt4 ? __uint_as_float((uint32_t) s4[i] << 16) : s8; }
};

// ---- one block ------------------------------------------------------------------------------------------------------------
// acc[i] += the product of the lane's rows g and g + 8 of the block (p) with the i-th eight rows of x, of which `live` are there.
// kMasked: x has rows of zeros that the weight is not meant for; `mask` names which of the lane's two columns may be added to: zero
// times a NaN is not zero.
//
// 8- and 4-bit weights as fp16.  x(i, term, q) gives octet q of row g of a term; scale(i, f, c) the scale of run f (FL = 64 or 128 long) of
// column 2 t + c.  A sum goes from scale to scale of the weight, then from scale to scale of x.
template <int FMT, int G, int FL, int NT, int kTerms, bool kMasked, typename X, typename R>
__device__ __forceinline__ void half_block(float (&acc)[NT][4], int live, const RowPiece<FMT> (&p)[2], const BlockScale<FMT, G> (&s)[2], unsigned mask, X &&x, R &&scale) {
    static_assert(FL == 64 || FL == 128, "an octet of 8-bit weights covers 64 neighbouring k");
    constexpr int kRun = G < FL ? G : FL;
    float c[NT][4], b[NT][4];
    uint32_t za[2] = {0, 0}, zb[2] = {0, 0};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int group = FMT == kWInt4 ? q * 32 / G : 0;
        const bool start = q % (kRun / 32) == 0, end = q % (kRun / 32) == kRun / 32 - 1, first = q % (FL / 32) < kRun / 32, last = q % (FL / 32) == FL / 32 - 1;
        if (FMT == kWInt4 && q * 32 % G == 0)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                za[h] = minus_zero(s[h].z4[group], 1024);
                zb[h] = minus_zero(s[h].z4[group], 64);
            }
        uint32_t wa[4], wb[4];
        p[0].halves(q, za[0], zb[0], wa);
        p[1].halves(q, za[1], zb[1], wb);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if (NT > 1 && i >= live) break;
            if (start) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.0f;
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
                const uint4 u = x(i, term, q);
                mma_16<__half>(c[i], wa[0], wb[0], wa[1], wb[1], u.x, u.y);
                mma_16<__half>(c[i], wa[2], wb[2], wa[3], wb[3], u.z, u.w);
            }
        }
        if (!end) continue;
        const float w[2] = {s[0].scale(group), s[1].scale(group)};
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if (NT > 1 && i >= live) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) b[i][j] = first ? c[i][j] * w[j >> 1] : b[i][j] + c[i][j] * w[j >> 1];
            if (!last) continue;
            const float xs[2] = {scale(i, q / (FL / 32), 0), scale(i, q / (FL / 32), 1)};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (!kMasked || (mask >> (j & 1) & 1)) acc[i][j] += b[i][j] * xs[j & 1];
        }
    }
}

// 16-bit weights.  x(i, term, q) gives octet q of row g of a term.
template <typename T, int NT, int kTerms, bool kMasked, typename X>
__device__ __forceinline__ void word_block(float (&acc)[NT][4], int live, const RowPiece<kW16> &pa, const RowPiece<kW16> &pb, unsigned mask, X &&x) {
    float c[NT][4] = {};
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if (NT > 1 && i >= live) break;
            float(&d)[4] = kMasked ? c[i] : acc[i];
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
                const uint4 u = x(i, term, q);
                mma_16<T>(d, pa.v[q].x, pb.v[q].x, pa.v[q].y, pb.v[q].y, u.x, u.y);
                mma_16<T>(d, pa.v[q].z, pb.v[q].z, pa.v[q].w, pb.v[q].w, u.z, u.w);
            }
        }
    if constexpr (kMasked)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (mask >> (j & 1) & 1) acc[i][j] += c[i][j];
}

__device__ __forceinline__ void split_half(const RowPiece<kW16> &p, RowPiece<kW16> &hi, RowPiece<kW16> &lo) {
#pragma unroll
    for (int v = 0; v < RowPiece<kW16>::kVecs; ++v) {
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
}

// ---- the walk over k ----------------------------------------------------------------------------------------------------
// WR x WK warps: WR neighbouring sets of 16 weight rows, WK shares of the blocks of k (share s takes blocks s, s + WK, ...).  The WR warps
// of a share use the same blocks of x, which they copy together; the shares do not wait for one another.
//
// In shared memory, per share and stage: kTerms * cols rows of 256 bytes of x, for scaled x the runs' scales [cols][128 / FL], then per
// warp 2 * kVecs * 512 bytes of weights.
template <int FMT, int FL, int WR, int WK> struct Walk {
    static constexpr int kThreads = 32 * WR * WK, kRows = 16 * WR; // of weight, per CTA
    static constexpr int kWarpBytes = 2 * RowPiece<FMT>::kVecs * 512, kRuns = kKB / FL;
    __host__ __device__ static constexpr int run_bytes(int cols) { return kScaledX<FMT> ? (cols * kRuns * 4 + 15) / 16 * 16 : 0; }
    __host__ __device__ static constexpr int stage_bytes(int terms, int cols) { return WR * kWarpBytes + terms * cols * 256 + run_bytes(cols); }
    // what the CTA's shared memory has to hold: the stages, then the sums of the shares
    template <int NT> static int smem(int stages, int terms, int cols) {
        const int a = stages * WK * stage_bytes(terms, cols), b = WK * NT * 8 * (kRows + 1) * 4;
        return a > b ? a : b;
    }
};

template <int WR> __device__ __forceinline__ void share_barrier(int share) {
    if constexpr (WR == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(share + 1), "n"(32 * WR) : "memory"); // barrier 0 is the CTA's
}

// src: row[h], scale[h]   first byte and scales of the lane's weight row g + 8 h
//      x(term, col)       where row `col` of x (of a plane) starts;   runs(col)  its scales
// K: length of a weight row; 16-bit rows of x end there too, a multiple of 8.
// Weights are fetched ahead of grid_dep_wait, x after it; then the kernel after this one may start (grid_dep_open).
// A block is few instructions' work, so the pointers of everything a lane copies are kept and moved on by constants.
template <typename T, int FMT, int G, int FL, int NT, int WR, int WK, int kStages, int kTerms, bool kSplit, typename Src>
__device__ __forceinline__ void few_rows_walk(float (&acc)[NT][4], uint8_t *smem, int K, int cols, int live, const Src &src) {
    using W = Walk<FMT, FL, WR, WK>;
    using Piece = RowPiece<FMT>;
    constexpr int kRowBytes = Piece::kVecs * 512, kStep = 2 * WR; // rows of x a share copies at a time
    constexpr int kXPasses = (kTerms * NT * 8 + kStep - 1) / kStep, kRunPasses = kScaledX<FMT> ? (NT * 8 * W::kRuns + 32 * WR - 1) / (32 * WR) : 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wr = warp % WR, share = warp / WR, blocks = (K + kKB - 1) / kKB;
    const bool ragged = K % kKB != 0;
    const int x_rows = kTerms * cols, x_bytes = x_rows * 256, stage_bytes = W::stage_bytes(kTerms, cols);
    const uint32_t base = shared_u32(smem) + share * kStages * stage_bytes, top = base + kStages * stage_bytes;
    const uint32_t w_at = x_bytes + W::run_bytes(cols) + wr * W::kWarpBytes + lane * 16;
    const int mine = blocks > share ? (blocks - share + WK - 1) / WK : 0;
    // A quarter of a warp reads two rows of x at once: the rows of a pair are shifted against each other so that it meets eight different
    // 16-byte banks (rows a lane copies are all even or all odd).
    constexpr int kShift = FMT == kWE4M3 || FMT == kWE5M2 ? 1 : 4;
    const int unit = lane & 15, x_first = wr * 2 + (lane >> 4), run_first = wr * 32 + lane;
    const uint32_t x_at = x_first * 256 + (unit ^ (x_first & 1) * kShift) * 16;

    const uint8_t *wp[2], *xp[kXPasses];
    const float *rp[kRunPasses > 0 ? kRunPasses : 1];
    int kb_w = share, kb_x = share;
    wp[0] = src.row[0] + (int64_t) share * Piece::kBlockBytes + t * 16;
    wp[1] = src.row[1] + (int64_t) share * Piece::kBlockBytes + t * 16;
    auto fetch_weights = [&](uint32_t slot) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (FMT == kWInt4 || !ragged || kb_w != blocks - 1) Piece::copy(slot + w_at + h * kRowBytes, wp[h]);
            else Piece::copy_last(slot + w_at + h * kRowBytes, wp[h], t, K - kb_w * kKB);
            wp[h] += WK * Piece::kBlockBytes;
        }
        kb_w += WK;
    };
    auto fetch_x = [&](uint32_t slot) {
#pragma unroll
        for (int i = 0; i < kXPasses; ++i)
            if (x_first + i * kStep < x_rows) {
                copy16(slot + x_at + i * (kStep * 256), xp[i], kScaledX<FMT> || !ragged || kb_x * kKB + unit * 8 < K);
                xp[i] += WK * 256;
            }
#pragma unroll
        for (int i = 0; i < kRunPasses; ++i)
            if (run_first + i * 32 * WR < cols * W::kRuns) {
                copy4(slot + x_bytes + (run_first + i * 32 * WR) * 4, rp[i]);
                rp[i] += WK * W::kRuns;
            }
        kb_x += WK;
    };
    BlockScale<FMT, G> s[2], next[2];
    RowScale<FMT> sp[2] = {src.scale[0], src.scale[1]};
    int kb_s = share;
    auto load_scales = [&] {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            next[h].load(sp[h], kb_s, kb_s == blocks - 1);
            BlockScale<FMT, G>::advance(sp[h], WK);
        }
        kb_s += WK;
    };
    if (mine > 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) BlockScale<FMT, G>::advance(sp[h], share);
        load_scales();
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i)
        if (i < mine) fetch_weights(base + i * stage_bytes);
    grid_dep_wait();
    grid_dep_open();
#pragma unroll
    for (int i = 0; i < kXPasses; ++i) {
        const int row = min(x_first + i * kStep, x_rows - 1), term = kTerms > 1 && row >= cols ? 1 : 0;
        xp[i] = src.x(term, row - term * cols) + (int64_t) share * 256 + unit * 16;
    }
#pragma unroll
    for (int i = 0; i < kRunPasses; ++i) {
        const int at = min(run_first + i * 32 * WR, cols * W::kRuns - 1);
        rp[i] = src.runs(at / W::kRuns) + share * W::kRuns + at % W::kRuns;
    }
    uint32_t fill = base, drain = base;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (i < mine) fetch_x(fill);
        copies_done();
        fill += stage_bytes;
    }
    // Where the lane finds its row of the i-th eight of x; a row that is not there reads another, its column is not looked at.
    uint32_t x_row[NT], x_odd[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int col = min(i * 8 + g, cols - 1);
        x_row[i] = col * 256;
        x_odd[i] = (col & 1) * kShift * 16;
    }
    const uint32_t term_bytes = cols * 256, term_odd = (cols & 1) * kShift * 16;
    for (int it = 0; it < mine; ++it) {
        copies_wait<kStages - 2>();
        share_barrier<WR>(share); // the block is there for every warp, and the stage before it is read by every warp
        if (it + kStages - 1 < mine) {
            fetch_weights(fill);
            fetch_x(fill);
            fill += stage_bytes;
            if (fill == top) fill = base;
        }
        copies_done();
        s[0] = next[0];
        s[1] = next[1];
        if (it + 1 < mine) load_scales();
        Piece p[2];
        p[0].read(drain + w_at);
        p[1].read(drain + w_at + kRowBytes);
        auto x = [&](int i, int term, int q) {
            const int at = FMT == kWE4M3 || FMT == kWE5M2 ? 128 * (q / 2) + 32 * t + 16 * (q % 2) : 64 * q + 16 * t;
            return read16(drain + x_row[i] + term * term_bytes + (at ^ x_odd[i] ^ (term * term_odd)));
        };
        if constexpr (kScaledX<FMT>) { // (a column that is not there reads what lies behind the runs)
            const uint32_t run_at = drain + x_bytes + 2 * t * W::kRuns * 4;
            half_block<FMT, G, FL, NT, kTerms, false>(acc, live, p, s, 3, x, [&](int i, int f, int c) { return read4(run_at + ((i * 8 + c) * W::kRuns + f) * 4); });
        } else if constexpr (!kSplit) {
            word_block<T, NT, kTerms, false>(acc, live, p[0], p[1], 3, x);
        } else { // fp16 weights become the sum of two bf16, exactly
            Piece ha, hb, la, lb;
            split_half(p[0], ha, la);
            split_half(p[1], hb, lb);
            word_block<T, NT, kTerms, false>(acc, live, ha, hb, 3, x);
            word_block<T, NT, 1, false>(acc, live, la, lb, 3, x);
        }
        drain += stage_bytes;
        if (drain == top) drain = base;
    }
    copies_wait<0>();
}

// The shares' sums in shared memory [share][column][row]: sum(column, row) adds them up, in the shares' order.
template <int NT, int WR, int WK> struct ShareSums {
    static constexpr int kPitch = 16 * WR + 1;
    float *part;
    __device__ __forceinline__ ShareSums(const float (&acc)[NT][4], uint8_t *smem) : part(reinterpret_cast<float *>(smem)) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        __syncthreads(); // the stages are read
        float *mine = part + (warp / WR) * (NT * 8) * kPitch + warp % WR * 16;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[(i * 8 + 2 * t + (j & 1)) * kPitch + g + (j >> 1) * 8] = acc[i][j];
        __syncthreads();
    }
    __device__ __forceinline__ float sum(int column, int row) const {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < WK; ++w) s += part[(w * NT * 8 + column) * kPitch + row];
        return s;
    }
};

// ---- scaling rows of x -------------------------------------------------------------------------------------------------------
struct ScaledRows { // planes [rows][pitch] of fp16, scales [rows][blocks * 128 / FL]
    uint8_t *planes;
    int64_t plane;  // bytes from plane to plane
    int64_t pitch;  // bytes of a row
    float *runs;
    int blocks;
};
inline int64_t scaled_bytes(int terms, int64_t rows, int64_t K, int FL) {
    const int64_t blocks = cdiv<int64_t>(K, kKB);
    return rows * blocks * (terms * kKB * 2 + kKB / FL * 4);
}
inline ScaledRows scaled_rows_at(void *p, int terms, int64_t rows, int64_t K) {
    const int64_t blocks = cdiv<int64_t>(K, kKB), pitch = blocks * kKB * 2;
    return {(uint8_t *) p, rows * pitch, pitch, (float *) ((uint8_t *) p + terms * rows * pitch), (int) blocks};
}

// The lane's four neighbouring values of a block of a row, zero past its end.
template <typename T> __device__ __forceinline__ void load_four(const T *x, int K, int k, float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = 0.0f;
    if (k >= K) return; // K is a multiple of 8
    if constexpr (sizeof(T) == 4) {
        const float4 u = *reinterpret_cast<const float4 *>(x + k);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(x + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_f32(reinterpret_cast<const T *>(&u)[j]);
    }
}
__device__ __forceinline__ float largest_of(const float (&v)[4], bool &fine) {
    float largest = 0.0f;
    fine = true;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float m = fabsf(v[j]);
        if (m < INFINITY) largest = fmaxf(largest, m);
        else fine = false;
    }
    return warp_max(largest);
}

// A warp scales a block, four values a lane, to fp16: `to` is the block's place in the first plane.
template <int FMT, int kTerms> __device__ __forceinline__ void scale_to_half(const float (&v)[4], uint8_t *to, int64_t plane, float *run) {
    const int lane = threadIdx.x & 31;
    bool fine;
    float scale, inv;
    block_scale(largest_of(v, fine), kTopHalf, scale, inv);
#pragma unroll
    for (int term = 0; term < kTerms; ++term) {
        __half h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = v[j] * inv;
            h[half_place<FMT>(j)] = term == 0 ? __float2half_rn(x) : __float2half_rn(fabsf(x) < INFINITY ? x - __half2float(__float2half_rn(x)) : 0.0f);
        }
        uint2 u;
        memcpy(&u, h, 8);
        *reinterpret_cast<uint2 *>(to + term * plane + lane * 8) = u;
    }
    if (lane == 0) *run = scale;
}

template <typename T, int FMT> __device__ __forceinline__ void scale_block(const T *x, int K, int kb, int64_t row, const ScaledRows &out) {
    float v[4];
    load_four(x, K, kb * kKB + (threadIdx.x & 31) * 4, v);
    scale_to_half<FMT, 1>(v, out.planes + row * out.pitch + kb * (kKB * 2), out.plane, out.runs + row * out.blocks + kb);
}

template <typename T, int FMT> __global__ void __launch_bounds__(128) scale_rows_kernel(const T *x, int64_t ldx, int M, int K, const ScaledRows out) {
    grid_dep_wait();
    grid_dep_open();
    const int blocks = (K + kKB - 1) / kKB, i = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i >= M * blocks) return;
    const int row = i / blocks;
    scale_block<T, FMT>(x + row * ldx, K, i - row * blocks, row, out);
}

} // namespace
} // namespace ptb
