// Products of a few rows of activations with a large weight, out[m, n] = sum_k x[m, k] * w[n, k], for weights of 16, 8 or 4 bits:
// what the 4-bit product and the MoE layer for few tokens share.
//
// Such a product reads the weight once and does little with it, so it is bound by HBM, and everything here serves to have
// many wide loads in flight and few instructions per weight.  The weight takes the 16-row side of mma.sync and eight rows of x the
// other: tcgen05 wants 128 weight rows, unpacked, in shared or tensor memory, which at one to sixteen rows buys nothing but a copy (for more it may pay; it
// has not been built).  A warp walks 128-wide blocks of k; its weights come as tensor boxes into two slots of its own, which it fills again as soon as it has
// read them.  No barrier of the CTA stands in the walk.
//
// What an MMA is fed with.  Measured on a B200, an SM issues an m16n8k16 of 16-bit floats or an m16n8k32 of bytes every 2.1 clocks (FP8
// ones are taken apart into these: 5.6), and integer and conversion instructions at 64 lanes a clock; HBM brings 23 bytes a clock
// and SM.  Unpacking 4-bit codes to bf16 is 7 such instructions for 8 codes, FP8 to bf16 8 for 4 values: too near the budget or beyond it.  So
//   * for a token or a few (few_tokens_walk) 4-bit codes go in as the bytes they are: two ANDs and a shift for 8 codes.  x is an integer
//     of three bytes, the first signed, scaled by a power of two per block that brings the largest of its 128 to 2^21 .. 2^22.  bf16's eight bits are
//     exact in it down to 2^-14 of the largest, fp16's eleven to 2^-11; below, a value is off by up to 2^-22 of the largest.  (With two bytes 2^-15: beside
//     an outlier of 1000 the result of the others is off by more than bf16's own rounding.  The third costs 3 %: 4096 x 14336, one row, 12.1 instead of
//     11.7 us, and room: rows that no longer fit are for the other walk, 2 rows of 14336 19.5 instead of 13.5.)  Sums of
//     a group are exact integers, and scaling them is what costs: with more columns of x than eight it is too much;
//   * for more (few_rows_walk) codes become fp16 less their zero, exactly, 9 instructions for 8.  That is what bounds it: 48 tokens through 32
//     experts of 7168 x 2048, groups of 32, 357 us where the weights' 790 MB are 121, with two thirds of all issue slots used.  Of these, scaling
//     the sums of the groups and their MMAs are a fifth, unpacking an eighth, fetching scales a tenth;
//   * FP8 weights are converted to fp16, exactly, one instruction for two;
//   * x goes with fp16 weights as fp16, scaled by a power of two per block into its range, where bf16 and fp16 values are exact down
//     to 2^-27 of the block's largest;
//   * 16-bit weights go in with 16-bit x as they are.
//
// The order of k inside an MMA is free as long as both operands agree on it.  Lane (g, t) = (lane / 4, lane % 4) of a warp supplies two weight
// rows (lane_row() and the eighth after it) and row g of x.  An "octet" is eight neighbouring k of a lane: one MMA of bytes, or two of 16
// bits.  A block of 128 is four octets a lane.  Where octet q of lane t lies:
//   16-bit and 4-bit weights  k = 32 q + 8 t                    (octet q of all four lanes: 32 neighbouring k, the smallest 4-bit group)
//   8-bit weights             k = 64 (q / 2) + 16 t + 8 (q % 2) (16 bytes a lane and load; octets 2 c and 2 c + 1: 64 neighbouring k)
#pragma once

#include "ptb_common.cuh"

#include <cuda.h>

#include <type_traits>

namespace ptb {
namespace {

enum WeightFormat { kW16 = 0, kWE4M3 = 1, kWE5M2 = 2, kWInt4 = 3 };
constexpr int kKB = 128; // k per block
template <int FMT> constexpr bool kScaledX = FMT != kW16; // x is scaled per block

// 4-bit weights.  Row n of a [N, K] weight is ceil(K / 128) blocks of 64 bytes.  Word t * 4 + q of a block holds octet (q, t), so lane t
// of a quad reads its four octets as one 16-byte piece.  Byte i of a word holds code i of the eight in its low nibble and code
// i + 4 in its high one.  Codes past K are 0.   value = (code - zero) * scale with any byte as zero, 8 where no zero points are given.
constexpr int kInt4BlockBytes = 64;
__device__ __forceinline__ int int4_shift(int i) { return (i & 3) * 8 + (i >> 2) * 4; } // of code i of a word

// ---- launches that start under the kernel before ----------------------------------------------------------------------
// A kernel that is launched with launch_early may start once every CTA of the kernel before has called grid_dep_open.  That one calls it
// after its own grid_dep_wait: so when a CTA of this kernel runs, everything before the kernel before is done, and what does not come
// from that kernel -- the weights -- may be fetched ahead of grid_dep_wait.  Every CTA calls grid_dep_wait before it leaves.
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dep_open() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Shared memory: `smem` for this launch, `most` for any.  The limit that is set belongs to the kernel, not to the launch, and another thread may launch
// the same kernel with other sizes between the two calls here: so it is the same number every time.
template <typename... P, typename... A>
inline cudaError_t launch_early(void (*kernel)(P...), dim3 grid, unsigned threads, int smem, int most, cudaStream_t st, unsigned cluster, A &&...args) {
    if (smem > most) return cudaErrorInvalidValue;
    if (smem > 32 * 1024) // 48 KB without asking, with what the kernel has besides
        if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) return e;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {cluster, 1, 1};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = (size_t) smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

inline int sm_count(int *sms) {
    int dev = 0;
    PTB_CUDA(cudaGetDevice(&dev));
    PTB_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    return 0;
}

// ---- copies -------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t shared_u32(const void *p) { return (uint32_t) __cvta_generic_to_shared(p); }
__device__ __forceinline__ uint4 read16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void zero16(uint32_t at) { asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory"); }
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
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_end(uint32_t bar) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
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
__device__ __forceinline__ void box_copy(uint32_t dst, const CUtensorMap *map, int byte, int row, int slab, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(byte), "r"(row), "r"(slab)
                 : "memory");
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
// c = a * b
__device__ __forceinline__ void mma_16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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
constexpr int kTopInt = 21, kTopHalf = 13;
// Where value k of a block stands: among the bytes that go with byte codes (lane t's four octets are 32 neighbouring bytes), and among the
// fp16 of the walk over rows (octet q of the four lanes: 64 neighbouring bytes; with 4-bit weights an octet's order is 0 2 1 3 4 6 5 7).
__host__ __device__ __forceinline__ int byte_place(int k) { return (k / 8 % 4) * 32 + (k / 32) * 8 + k % 8; }
template <int FMT> __host__ __device__ __forceinline__ int half_place(int k) {
    return FMT == kWInt4 ? (k & ~3) | (k & 1) << 1 | (k & 2) >> 1 : (k & ~63) | (k & 8) << 2 | (k & 48) >> 1 | (k & 7);
}

// ---- weights in shared memory ---------------------------------------------------------------------------------------------------
// A weight travels in chunks of 256 bytes of 16 rows: two boxes of 128 bytes (one to four blocks), which one thread asks for.  (As sixteen bulk copies, a
// row each, a chunk cost the warp 20 instructions a copy: an FP8 layer took 82 instead of 63 us.)  Past the end of a row a box is filled with zeros.  The
// 16-byte units of row r lie in the order unit ^ r % 8.  A quarter of a warp reads four units of two rows at once: rows r and r + 4 meet
// different banks, so lanes 4 g to 4 g + 3 have row g / 2 + 4 (g % 2) of a tile, and the row 8 further on.
constexpr int kBoxBytes = 16 * 128, kSlotBytes = 2 * kBoxBytes;
__device__ __forceinline__ int lane_row() {
    const int g = (threadIdx.x & 31) >> 2;
    return g >> 1 | (g & 1) << 2;
}
__device__ __forceinline__ uint32_t lane_place() { // of unit t of the row
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    return lane_row() * 128 + (g & 1) * 64 + (t ^ g >> 1) * 16;
}
// slabs of `rows` rows; a tile is 16 rows, or 8 rows of each of two neighbouring slabs
inline int weight_map(CUtensorMap *map, const void *data, int64_t row_bytes, int64_t rows, int64_t slabs, bool two) {
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                               CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = nullptr;
    if (encode == nullptr) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        PTB_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found));
        PTB_REQUIRE(found == cudaDriverEntryPointSuccess && p != nullptr, PTB_ERR_DRIVER, "cuTensorMapEncodeTiled is not available in this driver");
        encode = (Encode) p;
    }
    const cuuint64_t dims[3] = {(cuuint64_t) row_bytes, (cuuint64_t) rows, (cuuint64_t) slabs}, strides[2] = {(cuuint64_t) row_bytes, (cuuint64_t) (row_bytes * rows)};
    const cuuint32_t box[3] = {128, two ? 8u : 16u, two ? 2u : 1u}, steps[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(data), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    PTB_REQUIRE(r == CUDA_SUCCESS, PTB_ERR_DRIVER, "cuTensorMapEncodeTiled failed with CUresult %d", (int) r);
    return 0;
}
// Dynamic shared memory from where boxes may lie; kernels ask for kAlign bytes more.
constexpr int kAlign = 1024;
__device__ __forceinline__ uint8_t *aligned(uint8_t *smem) { return smem + (-shared_u32(smem) & (kAlign - 1)); }

// ---- one weight row's share of a lane in a block ----------------------------------------------------------------------
template <int FMT> struct RowPiece {
    static constexpr int kVecs = FMT == kWInt4 ? 1 : FMT == kW16 ? 4 : 2;
    uint4 v[kVecs];
    static constexpr int kBlockBytes = FMT == kWInt4 ? kInt4BlockBytes : FMT == kW16 ? 256 : 128;
    // block i of a chunk; at: the lane's place in the slot, `down` bytes on
    __device__ __forceinline__ void read(uint32_t at, int i, int down) {
        if constexpr (FMT == kWInt4) v[0] = read16(((at + (i >> 1) * kBoxBytes) ^ (i & 1) * 64) + down);
        else
#pragma unroll
            for (int j = 0; j < kVecs; ++j) v[j] = read16(((at + (FMT == kW16 ? j >> 1 : i) * kBoxBytes) ^ (j & 1) * 64) + down);
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
constexpr int kChunkRow = 256, kWeightSlots = 2; // slots of a warp
template <int FMT> constexpr int kChunk = kChunkRow / RowPiece<FMT>::kBlockBytes; // blocks

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
// One block's, packed as they are stored.  A lane asks for one block of a chunk, a chunk ahead, and the quad that shares the rows passes
// them round.
template <int FMT, int G> struct BlockScale {
    static constexpr int kN = FMT == kWInt4 ? kKB / G : 1, kWords = FMT == kWInt4 ? (kN + 1) / 2 : 1;
    uint32_t s[kWords], z;
    // the row's scales of block kb; zeros where there are none (there x and the codes are zero)
    __device__ __forceinline__ void load(const RowScale<FMT> &r, int kb, int blocks) {
        if constexpr (FMT == kWInt4) {
            if (kN > 1 && kb * kN + kN <= r.count && reinterpret_cast<uintptr_t>(r.s4 + kb * kN) % (2 * kN) == 0 && (r.z4 == nullptr || reinterpret_cast<uintptr_t>(r.z4 + kb * kN) % kN == 0)) {
                if constexpr (kN == 4) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(r.s4 + kb * kN);
                    s[0] = v.x;
                    s[kWords - 1] = v.y;
                    z = r.z4 != nullptr ? *reinterpret_cast<const uint32_t *>(r.z4 + kb * kN) : 0x08080808u;
                } else {
                    s[0] = *reinterpret_cast<const uint32_t *>(r.s4 + kb * kN);
                    z    = r.z4 != nullptr ? *reinterpret_cast<const uint16_t *>(r.z4 + kb * kN) : 0x0808u;
                }
                return;
            }
            z = 0;
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int at     = kb * kN + i;
                const bool there = at < r.count;
                const uint32_t v = there ? r.s4[at] : 0u;
                s[i / 2]         = i % 2 ? s[i / 2] | v << 16 : v;
                z |= (there && r.z4 != nullptr ? (uint32_t) r.z4[at] : 8u) << (8 * i);
            }
        } else if constexpr (FMT != kW16) {
            s[0] = kb < blocks ? __float_as_uint(r.s8[(int64_t) kb * r.stride]) : 0u;
        }
    }
    __device__ __forceinline__ BlockScale from_lane(int lane) const {
        BlockScale o;
        if constexpr (FMT != kW16)
#pragma unroll
            for (int i = 0; i < kWords; ++i) o.s[i] = __shfl_sync(0xffffffffu, s[i], lane);
        if constexpr (FMT == kWInt4) o.z = __shfl_sync(0xffffffffu, z, lane);
        return o;
    }
    __device__ __forceinline__ float scale(int i) const {
        if constexpr (FMT != kWInt4) return __uint_as_float(s[0]);
        return __uint_as_float(i % 2 ? s[i / 2] & 0xffff0000u : s[i / 2] << 16);
    }
    // -(1024 + zero) and -(64 + zero) in both halves, exact for every byte: fp16 numbers whose last bit is worth 1
    __device__ __forceinline__ void minus_zero(int i, uint32_t &za, uint32_t &zb) const {
        za = __byte_perm(z, 0, 0x4040 | i | i << 8) + 0xe400e400u;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(zb) : "r"(za), "r"(0x63806380u)); // plus 960
    }
};

// ---- one block ------------------------------------------------------------------------------------------------------------
// acc[i] += the product of the lane's rows g and g + 8 of the block (p) with the i-th eight rows of x, of NT.
//
// 8- and 4-bit weights as fp16.  x(i, term, q) gives octet q of row g of a term; scale(i, f, c) the scale of run f (FL = 64 or 128 long) of
// column 2 t + c.  A sum goes from scale to scale of the weight, then from scale to scale of x.
template <int FMT, int G, int FL, int NT, int kTerms, int kMost, typename X, typename R>
__device__ __forceinline__ void half_block(float (&acc)[kMost][4], const RowPiece<FMT> (&p)[2], const BlockScale<FMT, G> (&s)[2], bool zeros, X &&x, R &&scale) {
    static_assert(FL == 64 || FL == 128, "an octet of 8-bit weights covers 64 neighbouring k");
    constexpr int kRun = G < FL ? G : FL;
    float c[NT][4], b[NT][4];
    uint32_t za[2] = {0xe408e408u, 0xe408e408u}, zb[2] = {0xd480d480u, 0xd480d480u}; // of zero points of 8
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int group = FMT == kWInt4 ? q * 32 / G : 0;
        const bool start = q % (kRun / 32) == 0, end = q % (kRun / 32) == kRun / 32 - 1, first = q % (FL / 32) < kRun / 32, last = q % (FL / 32) == FL / 32 - 1;
        if (FMT == kWInt4 && q * 32 % G == 0 && zeros)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h].minus_zero(group, za[h], zb[h]);
        uint32_t wa[4], wb[4];
        p[0].halves(q, za[0], zb[0], wa);
        p[1].halves(q, za[1], zb[1], wb);
        const float w[2] = {s[0].scale(group), s[1].scale(group)};
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
                const uint4 u = x(i, term, q);
                if (start && term == 0) mma_16_first(c[i], wa[0], wb[0], wa[1], wb[1], u.x, u.y);
                else mma_16<__half>(c[i], wa[0], wb[0], wa[1], wb[1], u.x, u.y);
                mma_16<__half>(c[i], wa[2], wb[2], wa[3], wb[3], u.z, u.w);
            }
        }
        if (!end) continue;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) b[i][j] = first ? c[i][j] * w[j >> 1] : b[i][j] + c[i][j] * w[j >> 1];
            if (!last) continue;
            const float xs[2] = {scale(i, q / (FL / 32), 0), scale(i, q / (FL / 32), 1)};
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] += b[i][j] * xs[j & 1];
        }
    }
}

// 16-bit weights.  x(i, term, q) gives octet q of row g of a term.
template <typename T, int NT, int kTerms, int kMost, typename X>
__device__ __forceinline__ void word_block(float (&acc)[kMost][4], const RowPiece<kW16> &pa, const RowPiece<kW16> &pb, X &&x) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
                const uint4 u = x(i, term, q);
                mma_16<T>(acc[i], pa.v[q].x, pb.v[q].x, pa.v[q].y, pb.v[q].y, u.x, u.y);
                mma_16<T>(acc[i], pa.v[q].z, pb.v[q].z, pa.v[q].w, pb.v[q].w, u.z, u.w);
            }
        }
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
// WR warps, each with 16 weight rows and two slots of chunks of its own, which it fills again as soon as it has read them.  x is shared: a
// ring of two pairs of blocks.  A warp that has read a pair says so, and goes on; once it has read the first block of the next, one warp, each in its turn,
// waits for all to have said so and copies the pair after that there.
//
// Rows of x are shifted against each other so that a quarter of a warp, two rows at once, meets different banks.  Scaled x is
// stored with its scales: 256 bytes of a block, then the scales of its runs.
constexpr int kScaledBlock = 256 + 16, kPair = 2, kXPitch = kPair * 256 + 64;
template <int FMT, int NT, int WR> struct Walk {
    static constexpr int kThreads = 32 * WR, kRows = 16 * WR; // rows of the weight
    static constexpr int kXStep = kScaledX<FMT> ? kScaledBlock : 256;
    static constexpr int kBars = WR * kWeightSlots + 2 * kPair;
    static constexpr int kSums = NT * 8 * (kRows + 1) * 4;
    // what the CTA's shared memory has to hold: the slots and the ring, read to the end of eight columns, then the sums and `more`
    static constexpr int smem(int terms, int cols, int more = 0) {
        const int a = WR * kWeightSlots * kSlotBytes + (2 * terms * cols + 7) * kXPitch, b = kSums + more;
        return (a > b ? a : b) + kAlign;
    }
};

template <int FMT> struct LaneRows { // the warp's tile in the weight's map, and the scales of rows lane_row() and lane_row() + 8
    int row, slab;
    RowScale<FMT> scale[2];
};
// n blocks of a tile from block kb on into a slot, by one thread
template <int FMT> __device__ __forceinline__ void fetch_tile(uint32_t slot, const CUtensorMap *map, int kb, int n, int row, int slab, uint32_t bar) {
    constexpr int kBytes = RowPiece<FMT>::kBlockBytes;
    const int boxes = (n * kBytes + 127) / 128;
    bar_expect(bar, boxes * kBoxBytes);
    box_copy(slot, map, kb * kBytes, row, slab, bar);
    if (boxes > 1) box_copy(slot + kBoxBytes, map, kb * kBytes + 128, row, slab, bar);
}

// body(the number of eights of x as a constant): branches on it in the middle of a block cost ten instructions each.
template <int NT, typename F> __device__ __forceinline__ void by_live(int live, F &&body) {
    if constexpr (NT > 1)
        if (live < NT) return by_live<NT - 1>(live, body);
    body(std::integral_constant<int, NT>{});
}

// src: a LaneRows, and x(term, col): where row `col` of x (of a plane) starts.  [begin, end): blocks of k, begin at the start of a chunk.
// K: length of a weight row; 16-bit rows of x end there too.
// Weights are fetched ahead of grid_dep_wait, x after it; then the kernel after this one may start (grid_dep_open).
// Called by all threads; what the shared memory held is read, and the barriers are free again, when it returns.
template <typename T, int FMT, int G, int FL, int NT, int WR, int kTerms, bool kSplit, typename Src>
__device__ __forceinline__ void few_rows_walk(float (&acc)[NT][4], uint8_t *smem, uint64_t *bars, const CUtensorMap *map, int K, int cols, int begin, int end, const Src &src) {
    using W = Walk<FMT, NT, WR>;
    using Piece = RowPiece<FMT>;
    constexpr int CB = kChunk<FMT>;
    static_assert(kTerms * NT <= WR && (WR & (WR - 1)) == 0, "the warps copy eight rows of x each");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int live = (cols + 7) / 8, x_rows = kTerms * cols, x_warps = (x_rows + 7) / 8;
    const uint32_t ring = shared_u32(smem) + warp * (kWeightSlots * kSlotBytes), x_ring = shared_u32(smem) + WR * (kWeightSlots * kSlotBytes), x_stage = x_rows * kXPitch;
    const uint32_t w_bars = shared_u32(bars) + warp * (kWeightSlots * 8), x_bars = shared_u32(bars) + WR * (kWeightSlots * 8), read_bars = x_bars + 2 * 8;
    if (threadIdx.x < W::kBars) bar_init(shared_u32(bars) + threadIdx.x * 8, (int) threadIdx.x < WR * kWeightSlots ? 1 : threadIdx.x < W::kBars - 2 ? x_warps : WR);
    bar_init_fence();
    __syncthreads();

    // Whole pairs are read: where the last has one block, the other is zeros.
    const int pairs = (end - begin + kPair - 1) / kPair;
    int kb_w = begin;
    auto fetch_weights = [&](int slot) {
        if (kb_w < begin + pairs * kPair && lane == 0)
            fetch_tile<FMT>(ring + slot * kSlotBytes, map, kb_w, min(CB, begin + pairs * kPair - kb_w), src.row, src.slab, w_bars + slot * 8);
        kb_w += CB;
    };
    BlockScale<FMT, G> next[2], mine[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) next[h].load(src.scale[h], begin + t, CB > 1 || t == 0 ? end : 0);
#pragma unroll
    for (int i = 0; i < kWeightSlots; ++i) fetch_weights(i);
    grid_dep_wait();
    grid_dep_open();
    // By the warps in turn, eight rows each: a copy takes a warp some 60 clocks.
    auto fetch_x = [&](int pair, auto &&free) {
        const int turn = (warp - pair) & (WR - 1), row = turn * 8 + lane, kb = begin + pair * kPair, stage = pair & 1;
        if (turn >= x_warps || !free()) return;
        uint32_t bytes = kScaledX<FMT> ? min(kPair, end - kb) * kScaledBlock : min(kPair * kKB, K - kb * kKB) * 2;
        const uint32_t to = x_ring + stage * x_stage + row * kXPitch;
        const bool mine = lane < 8 && row < x_rows;
        if (mine) // zeros behind the end: the weights are zero there too, but what lies here might be a NaN
            for (uint32_t i = bytes; i < kPair * W::kXStep; i += 16) zero16(to + i);
        __syncwarp();
        if (lane == 0) bar_expect(x_bars + stage * 8, min(8, x_rows - turn * 8) * bytes);
        __syncwarp();
        if (mine) {
            const int term = kTerms > 1 && row >= cols ? 1 : 0;
            bulk_copy(to, src.x(term, row - term * cols) + (int64_t) kb * W::kXStep, bytes, x_bars + stage * 8);
        }
    };
#pragma unroll 1
    for (int i = 0; i < 2 && i < pairs; ++i) fetch_x(i, [] { return true; });

    const uint32_t w_lane = ring + lane_place();
    const uint32_t x_lane = x_ring + g * kXPitch + t * 16, run_lane = x_ring + 2 * t * kXPitch + 256, term_bytes = cols * kXPitch;
    int slot = 0;
    uint32_t w_parity = 0;
    bool ok = true;
    auto next_chunk = [&] {
        if (ok) ok = __all_sync(0xffffffffu, bar_wait(w_bars + slot * 8, w_parity));
    };
    auto chunk_read = [&] {
        __syncwarp();
        if (ok) fetch_weights(slot);
        if (++slot == kWeightSlots) { slot = 0; w_parity ^= 1; }
    };
#pragma unroll 1
    for (int pair = 0; pair < pairs; ++pair) {
        const int kb = begin + pair * kPair, stage = pair & 1, in = kb % CB; // in: blocks done of the chunk
        if (in == 0) {
            next_chunk();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mine[h] = next[h];
                next[h].load(src.scale[h], kb + CB + t, end);
            }
        }
        if (ok) ok = __all_sync(0xffffffffu, bar_wait(x_bars + stage * 8, pair >> 1 & 1));
        if (pair > 0 && pair + 1 < pairs) // the pair after this one
            fetch_x(pair + 1, [&] {
                if (ok) ok = __all_sync(0xffffffffu, bar_wait(read_bars + (stage ^ 1) * 8, (pair - 1) >> 1 & 1));
                return ok;
            });
        if (ok) {
            const uint32_t x_at = stage * x_stage;
            by_live<NT>(live, [&](auto n) {
                constexpr int N = decltype(n)::value;
#pragma unroll // (one piece of code: more to do while something is waited for)
                for (int u = 0; u < kPair; ++u) {
                    if (CB == 1 && u > 0) {
                        chunk_read();
                        next_chunk();
                    }
                    Piece p[2];
                    p[0].read(w_lane + slot * kSlotBytes, CB > kPair ? in + u : CB > 1 ? u : 0, 0);
                    p[1].read(w_lane + slot * kSlotBytes, CB > kPair ? in + u : CB > 1 ? u : 0, 8 * 128);
                    auto x = [&](int i, int term, int q) { return read16(x_lane + x_at + u * W::kXStep + i * (8 * kXPitch) + term * term_bytes + q * 64); };
                    if constexpr (kScaledX<FMT>) {
                        BlockScale<FMT, G> s[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) s[h] = mine[h].from_lane((lane & 28) | (CB > kPair ? in + u : u));
                        half_block<FMT, G, FL, N, kTerms>(acc, p, s, src.scale[0].z4 != nullptr, x,
                                                          [&](int i, int f, int c) { return read4(run_lane + x_at + u * W::kXStep + (i * 8 + c) * kXPitch + f * 4); });
                    } else if constexpr (!kSplit) {
                        word_block<T, N, kTerms>(acc, p[0], p[1], x);
                    } else { // fp16 weights become the sum of two bf16, exactly
                        Piece ha, hb, la, lb;
                        split_half(p[0], ha, la);
                        split_half(p[1], hb, lb);
                        word_block<T, N, kTerms>(acc, ha, hb, x);
                        word_block<T, N, 1>(acc, la, lb, x);
                    }
                }
            });
        }
        if (in + kPair >= CB || pair == pairs - 1) chunk_read();
        __syncwarp();
        if (lane == 0) bar_arrive(read_bars + stage * 8);
    }
    if (!ok) { // the result is incomplete; what is on its way lands before the CTA gives its memory back
        if (lane == 0) atomicExch(&g_few_status, 5);
        for (int i = 0; i < kWeightSlots; ++i) bar_wait(w_bars + i * 8, i < slot ? w_parity ^ 1 : w_parity);
        for (int i = max(pairs - 2, 0); i < pairs; ++i) bar_wait(x_bars + (i & 1) * 8, i >> 1 & 1);
    }
    __syncthreads();
    if (threadIdx.x < W::kBars) bar_end(shared_u32(bars) + threadIdx.x * 8);
}

// The CTAs of a cluster may share k, each a run of four blocks or more (whole chunks and pairs); each adds up a part of the results, in the order of k.
constexpr int kShareBlocks = 4;
struct Share {
    int begin, end; // blocks
};
__device__ __forceinline__ Share share_of(int K, int share, int shares) {
    const int blocks = (K + kKB - 1) / kKB, runs = (blocks + kShareBlocks - 1) / kShareBlocks;
    return {share * runs / shares * kShareBlocks, min(blocks, (share + 1) * runs / shares * kShareBlocks)};
}
// As many as it takes to give every place of the device a CTA.  Without: 64 rows, 8192 x 8192 in 4 bits (128 CTAs, 256 with), 83 instead of 49 us;
// an MoE layer of 16 tokens, 2 of 8 experts of 7168 x 256, 45 instead of 24 us.
inline int shares_for(int K, int64_t ctas, int places) {
    int shares = 1;
    while (shares < 8 && 2 * shares <= cdiv(K, kKB * kShareBlocks) && ctas * shares * 2 <= places) shares *= 2;
    return shares;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float read_peer(const float *p, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(shared_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// The sums in shared memory [column][row].
template <int FMT, int NT, int WR> struct RowSums {
    static constexpr int kPitch = Walk<FMT, NT, WR>::kRows + 1;
    float *part;
    __device__ __forceinline__ RowSums(const float (&acc)[NT][4], uint8_t *smem) : part(reinterpret_cast<float *>(smem)) {
        const int warp = threadIdx.x >> 5, t = threadIdx.x & 3;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[(i * 8 + 2 * t + (j & 1)) * kPitch + warp * 16 + lane_row() + (j >> 1) * 8] = acc[i][j];
        __syncthreads();
    }
    __device__ __forceinline__ float sum(int column, int row, int shares) const { // shares > 1: between two cluster_sync
        float *at = &part[column * kPitch + row], s = 0.0f;
        if (shares == 1) return *at;
        for (int r = 0; r < shares; ++r) s += read_peer(at, r);
        return s;
    }
};

// ---- scaling rows of x -------------------------------------------------------------------------------------------------------
struct ScaledRows { // [terms][rows][blocks] of 128 fp16 and, in the first term, the scales of the block's runs
    uint8_t *planes;
    int64_t plane; // bytes from term to term
    int64_t pitch; // bytes of a row
};
inline int64_t scaled_bytes(int terms, int64_t rows, int64_t K) { return terms * rows * cdiv<int64_t>(K, kKB) * kScaledBlock; }
inline ScaledRows scaled_rows_at(void *p, int64_t rows, int64_t K) {
    const int64_t pitch = cdiv<int64_t>(K, kKB) * kScaledBlock;
    return {(uint8_t *) p, rows * pitch, pitch};
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
__device__ __forceinline__ float largest_of(const float (&v)[4]) { // of the warp's finite ones
    float largest = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (fabsf(v[j]) < INFINITY) largest = fmaxf(largest, fabsf(v[j]));
    return warp_max(largest);
}

// Values k to k + 3 of a block, times inv, as fp16; or what that leaves.
template <int FMT> __device__ __forceinline__ void put_halves(uint8_t *block, int k, const float (&v)[4], float inv, bool rest) {
    __half h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float s = v[j] * inv;
        h[half_place<FMT>(j)] = !rest ? __float2half_rn(s) : __float2half_rn(fabsf(s) < INFINITY ? s - __half2float(__float2half_rn(s)) : 0.0f);
    }
    uint2 u;
    memcpy(&u, h, 8);
    *reinterpret_cast<uint2 *>(block + (half_place<FMT>(k) & ~3) * 2) = u;
}

// A warp scales block kb of a row, four values a lane.
template <typename T, int FMT> __device__ __forceinline__ void scale_block(const T *x, int K, int kb, int64_t row, const ScaledRows &out) {
    const int lane = threadIdx.x & 31;
    float v[4], scale, inv;
    load_four(x, K, kb * kKB + lane * 4, v);
    block_scale(largest_of(v), kTopHalf, scale, inv);
    uint8_t *to = out.planes + row * out.pitch + (int64_t) kb * kScaledBlock;
    put_halves<FMT>(to, lane * 4, v, inv, false);
    if (lane == 0) *reinterpret_cast<float *>(to + 256) = scale;
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
