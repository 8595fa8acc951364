// Microscaled 4-bit numbers (MXFP4 of the OCP microscaling formats): 32 neighbouring entries of a row share a power of two
// 2^(s - 127), s one byte (255: not a number), and are held as e2m1, a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.
//
// Quantisation of a block with largest magnitude a: s - 127 = max(floor(log2 a) - 2, -127), so that the largest entry lands in
// [4, 8) (6 is the most that e2m1 holds, 2 its largest exponent); code = e2m1(x 2^(127 - s)), nearest, ties to the even code, at
// most 6.  The product with the power of two is exact for every float32 that does not round to zero anyway, so the result
// is the same in any arithmetic that holds the inputs.  A block with an infinity or a NaN has s = 255 and codes 0.
//
// Layout.  Codes: [rows, k / 2] bytes, the even entry in the low half of its byte.  Scales: atoms of 512 bytes for 128 rows by 4
// blocks (128 entries along k), atom (row / 128, block / 4) with byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4: what
// tcgen05.cp.32x128b.warpx4 spreads over tensor memory for a block-scaled product.  The atoms of 128 rows lie in order of k, an
// even number of them, with zeros behind the last block, so that 256 entries along k are 1,024 contiguous bytes.
#pragma once
#include "common.cuh"

#define MX4_BLOCK 32
#define MX4_ATOM 512
#define MX4_CHUNK 256                        // entries along k of a stage: 128 bytes of codes, two atoms

__host__ __device__ __forceinline__ long long mx4_atoms_k(long long k) { return 2 * ((k + MX4_CHUNK - 1) / MX4_CHUNK); }
// byte of (row, block of 32) inside the scales of a matrix with kg atoms along k
__host__ __device__ __forceinline__ size_t mx4_scale_at(long long row, long long block, long long kg) {
    return (size_t)((row >> 7) * kg + (block >> 2)) * MX4_ATOM + (size_t)((row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3));
}

// The scale byte of a block from the bits of its largest magnitude (the largest of the magnitudes' bits: a NaN beats an
// infinity beats every number).
__device__ __forceinline__ uint32_t mx4_scale_of(uint32_t top_bits) {
    const uint32_t e = top_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// What the entries are multiplied by: 2^(127 - s); 0 for a block that is not a number.
__device__ __forceinline__ float mx4_inverse(uint32_t s) { return s == 255u ? 0.f : __uint_as_float((254u - s) << 23); }

// Eight entries as codes, the first in the lowest half byte.
__device__ __forceinline__ uint32_t mx4_encode8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// The bits of the largest magnitude among eight entries (a NaN's are above an infinity's, and those above every number's).
__device__ __forceinline__ uint32_t mx4_top8(const float (&v)[8]) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, __float_as_uint(v[i]) & 0x7fffffffu);
    return t;
}
__device__ __forceinline__ uint32_t mx4_top8(const uint4 u) {          // bfloat16, two a word
    const uint32_t m = 0x7fff7fffu;
    const uint32_t t = __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
    return max(t << 16, t & 0xffff0000u);
}

// The scale byte of a block whose four lanes' largest magnitudes are `top`, and in `word` the four scale bytes of the 128 entries of the
// lane's sixteen neighbours.
__device__ __forceinline__ uint32_t mx4_block_scale(uint32_t top, int lane, uint32_t& word) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t s = mx4_scale_of(top);
    word = s << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    return s;
}
// Eight neighbouring entries of one lane, the four lanes of a block side by side: their codes, and `word` as above.
__device__ __forceinline__ uint32_t mx4_quantize8(const float (&v)[8], uint32_t top, int lane, uint32_t& word) {
    const uint32_t s = mx4_block_scale(top, lane, word);
    const float inv = mx4_inverse(s);
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = v[i] * inv;
    const uint32_t code = mx4_encode8(w);
    return s == 255u ? 0u : code;
}

// Eight bfloat16 as float32.
__device__ __forceinline__ void mx4_unpack(const uint4 u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
// Eight neighbouring float32 (p 16-byte aligned for VEC).
template <bool VEC> __device__ __forceinline__ void mx4_load8(const float* p, float (&v)[8]) {
    if (VEC) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
}
