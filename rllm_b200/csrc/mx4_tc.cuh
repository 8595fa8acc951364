// Products of microscaled 4-bit numbers on tcgen05: the instructions' wrappers and the tensor map of codes, shared by the kernels
// for few and for many rows.
#pragma once
#include "tcgen05.cuh"
#include "mx4.cuh"

#define MX4_SF_BYTES (2 * MX4_ATOM)                        // the scales of 128 rows in a stage of 256 entries along K

// ---------------------------------------------------------------- the instructions
// Instruction descriptor of kind mxf4: A and B e2m1 (1), scales ue8m0 (bit 23), both operands K-major, shape M x N x 64; bits 4-5 and
// 29-30 say which bytes of the scale columns belong to B and A (0 or 2: two scales a row and instruction).
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, int sf_id) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) | ((uint32_t)sf_id << 4) |
           ((uint32_t)sf_id << 29);
}
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// Shared-memory descriptor of one atom of scales: 32 lines of 16 bytes without swizzle, groups of 8 lines 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_atom(uint32_t saddr) {
    return ((uint64_t)((128u >> 4) | (1u << 14)) << 32) | ((saddr & 0x3FFFFu) >> 4);
}
// 512 bytes -> four columns, the 32 lines repeated for the four quarters of the lanes
__device__ __forceinline__ void tmem_cp_atom(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// 8 and 16 columns of the warp's lanes
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(s_addr(dst)), "l"(src), "r"(bytes), "r"(s_addr(bar)) : "memory");
}

// ---------------------------------------------------------------- host side
// Tensor map of codes [rows, k / 2] (contiguous): boxes of box_rows x 128 bytes, 128-byte swizzle, zeros outside.
static int mx4_tmap(CUtensorMap* map, const void* base, long long rows, int k, int box_rows) {
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
