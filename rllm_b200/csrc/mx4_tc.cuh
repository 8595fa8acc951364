// Products of microscaled 4-bit numbers on tcgen05: the instructions' wrappers and the tensor map of codes, shared by the kernels
// for few and for many rows.
#pragma once
#include "tcgen05.cuh"
#include "mx4.cuh"
#include "asked_once.h"
#include <math.h>

#define MX4_SF_BYTES (2 * MX4_ATOM)                        // the scales of 128 rows in a stage of 256 entries along K

// ---------------------------------------------------------------- the instructions
// A role's whole warp runs its loop and one elected lane issues (the predicate `on` of the wrappers below): the loop's counters and addresses
// are then uniform over the warp and live in uniform registers, which is where these instructions take their operands from.  With the
// loop inside `if (lane == 0)` every operand is moved there first, and the eleven instructions of a stage took about 1,000 cycles to issue.
__device__ __forceinline__ uint32_t warp_elect() {
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on;
}
// mbar_wait by a whole warp with one answer
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const volatile int* abort_flag) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
// Instruction descriptor of kind mxf4: A and B e2m1 (1), scales ue8m0 (bit 23), both operands K-major, shape M x N x 64; bits 4-5 and
// 29-30 say which bytes of the scale columns belong to B and A (0 or 2: two scales a row and instruction).
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, int sf_id) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) | ((uint32_t)sf_id << 4) |
           ((uint32_t)sf_id << 29);
}
// Descriptors by their low words (upper words are constant): a K-major tile with 128-byte swizzle (smem_desc_sw128), and one atom of scales,
// 32 lines of 16 bytes without swizzle, groups of 8 lines 128 bytes apart.  Shared memory ends below 2^18, so an offset in 16-byte units may be
// added to a low word.
__device__ __forceinline__ uint32_t tile_lo(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t atom_lo(uint32_t saddr) { return (saddr & 0x3FFFFu) >> 4; }
__device__ __forceinline__ uint64_t tile_desc(uint32_t lo) { return ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32) | lo; }
__device__ __forceinline__ uint64_t atom_desc(uint32_t lo) { return ((uint64_t)((128u >> 4) | (1u << 14)) << 32) | lo; }

// CG: CTAs that work together (the instructions' cta_group)
template <int CG> __device__ __forceinline__ void umma_mxf4(uint32_t on, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                            uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(on) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
            "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(on) : "memory");
}
// 512 bytes -> four columns, the 32 lines repeated for the four quarters of the lanes (CG 2: in each CTA its own bytes)
template <int CG> __device__ __forceinline__ void tmem_cp_atom(uint32_t on, uint32_t taddr, uint64_t desc) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}"
                     ::"r"(taddr), "l"(desc), "r"(on) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}"
                     ::"r"(taddr), "l"(desc), "r"(on) : "memory");
}
// CG 2: arrives at the barrier at this offset in both CTAs
template <int CG> __device__ __forceinline__ void umma_done(uint32_t on, uint64_t* bar) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                     "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                     ::"r"(s_addr(bar)), "r"(on) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                     "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}"
                     ::"r"(s_addr(bar)), "r"(on), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void warp_expect_tx(uint32_t on, uint64_t* bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}"
                 ::"r"(s_addr(bar)), "r"(bytes), "r"(on) : "memory");
}
__device__ __forceinline__ void warp_load_2d(uint32_t on, uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
        ::"r"(dst), "l"(map), "r"(s_addr(bar)), "r"(x), "r"(y), "r"(on) : "memory");
}
// the bytes complete on a barrier given by its cluster address (the leader's)
__device__ __forceinline__ void warp_load_2d_pair(uint32_t on, uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(on) : "memory");
}
__device__ __forceinline__ void warp_bulk_load(uint32_t on, uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
                 "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(s_addr(bar)), "r"(on) : "memory");
}
// 16 columns of the warp's lanes
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr) : "memory");
}

// C += v where the sum is made, in L2: nobody waits for the old value (an element gets one addition a launch, so the result does not depend on any
// order; a sum below 2^-126 becomes zero).  2,048 x 4,096 x 4,096: 49 us with loads and stores, 26 with these, 25 where C is only written.
__device__ __forceinline__ void add_to(float* p, float v) { asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(p), "f"(v) : "memory"); }
__device__ __forceinline__ void add_to4(float* p, const uint4 v) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};"
                 ::"l"(p), "f"(__uint_as_float(v.x)), "f"(__uint_as_float(v.y)), "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w)) : "memory");
}

// The gated unit of common.cuh's GluForm with the reciprocal of the special-function unit (1 ulp) in place of a division.  The denominator is taken by
// a quarter, and so is c: 1 + e^-z reaches 2^128, the reciprocal of more than 2^126 would be a subnormal number, and zero; so every finite one has its own
// (where the exponential is infinite the result is 0, as in common.cuh).  Gated 2,048 x 2 x 12,288 x 4,096: 85.2 us, with __fdividef, which gives 0 beyond
// 2^126, 85.0.  What the form asks is decided once: no clamp is a clamp at infinity, and the tanh form of gelu (alpha 0) a function of its own.  The
// clamps leave a NaN what it is.  (With the questions asked for every element a tile of 128 x 256 took 1.9 us longer to end.)
struct Mx4Glu {
    float limit, alpha, shift;
    bool gelu;
    __device__ __forceinline__ explicit Mx4Glu(const GluForm& f)
        : limit(f.limit > 0.f ? f.limit : INFINITY), alpha(f.alpha), shift(f.shift), gelu(f.alpha == 0.f) {}
    template <bool GELU> __device__ __forceinline__ float at(float g, float u) const {
        float c;
        asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(g), "f"(limit));
        asm("min.NaN.f32 %0, %1, %2;" : "=f"(u) : "f"(u), "f"(limit));
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(u) : "f"(u), "f"(-limit));
        const float z = GELU ? 1.5957691216057308f * (c + 0.044715f * c * c * c) : alpha * c;
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(0.25f, __expf(-z), 0.25f)));
        return 0.25f * c * r * (u + shift);
    }
};

// ---------------------------------------------------------------- host side
// Lets a kernel have `bytes` of dynamic shared memory on the current device; asked of the runtime once for each of them.
template <typename F> static int mx4_allow_smem(F* kern, int bytes) {
    static AskedOnce* const table = new AskedOnce;       // (never destroyed: threads may still launch while the process ends)
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    return table->once((const void*)kern, dev,
                       [&] { return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
}

// Tensor map of codes [rows, k / 2] (contiguous): boxes of box_rows x 128 bytes, 128-byte swizzle, zeros outside.
static inline int mx4_tmap(CUtensorMap* map, const void* base, long long rows, int k, int box_rows) {
    TmapEncodeFn enc = tmap_encoder();
    if (!enc) return 30001;
    const cuuint64_t dims[2] = {(cuuint64_t)(k / 2), (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(k / 2)};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 30000 + (int)r;
}

// Tensor map of scales: `lines` of 1,024 bytes (128 rows by 256 entries along K each), a line a box.
static inline int mx4_scale_tmap(CUtensorMap* map, const void* base, long long lines) {
    TmapEncodeFn enc = tmap_encoder();
    if (!enc) return 30001;
    const cuuint64_t dims[2] = {256, (cuuint64_t)lines};
    const cuuint64_t strides[1] = {MX4_SF_BYTES};
    const cuuint32_t box[2] = {256, 1}, estr[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 30000 + (int)r;
}
