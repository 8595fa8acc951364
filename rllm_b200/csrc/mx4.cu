// Rows to microscaled 4-bit numbers and back (mx4.cuh has the format and its layout).
//
//   mx4_quantize    codes and scales of the rows of x [rows, k] (float32 or bfloat16, any row stride).  With `offsets` the rows are
//                   those of routed experts: x has a row per token (`place` given: pair p of token p / top_k goes to row
//                   place[p] of the sorted rows) or the sorted rows themselves, and the scales lie in the order of the products'
//                   row tiles: expert e's rows begin a new block of 128 scale rows, the one behind the blocks of the experts before it.
//   mx4_dequantize  the values that codes and scales stand for, exact in float32 and in bfloat16.
//
// Both read and write every byte once; a warp takes 256 neighbouring entries of a row, a lane eight of them, so that loads are
// 512 or 1,024 and code stores 128 contiguous bytes; the four lanes of a block find its largest magnitude with two shuffles.
#include "mx4.cuh"

template <typename T, bool VEC, bool SORTED>
__global__ void __launch_bounds__(128)
mx4_quantize_kernel(const T* x, long long ld, int rows, int k, uint8_t* codes, uint8_t* scales, int pad_rows,
                    const int* offsets, const int* place, int E, int top_k) {
    // the kernels behind may start once the ones before are complete: a product reads its weights ahead of its own wait, and
    // those may be what the kernel before this one wrote
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int chunks = (k + MX4_CHUNK - 1) / MX4_CHUNK;
    const long long kg = 2 * (long long)chunks;
    const long long n_warps = (long long)gridDim.x * (blockDim.x >> 5);
    for (long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < (long long)pad_rows * chunks; w += n_warps) {
        const long long item = w / chunks;
        const int c = (int)(w - item * chunks), col = c * MX4_CHUNK + lane * 8;
        long long src = item, row = item, scale_row = item;
        if (SORTED) {
            if (place) {
                row = place[item];
                src = item / top_k;
                if (row < 0 || row >= rows) continue;
            }
            // the row's expert: the last one that begins at or before it; and the row tiles of the experts before that one
            int lo = 0, hi = E;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (offsets[mid] <= row) lo = mid; else hi = mid;
            }
            int tiles = 0;
            for (int e = lane; e < lo; e += 32) tiles += (offsets[e + 1] - offsets[e] + 127) >> 7;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
            scale_row = (long long)tiles * 128 + (row - offsets[lo]);
            // (offsets that do not rise from 0 to the number of rows: nothing outside the scales is written)
            if (scale_row < 0 || scale_row >= ((long long)((rows + 127) >> 7) + E) * 128) continue;
        }
        float v[8];
        const bool in = item < rows && col < k;                  // (k is a multiple of 32: a lane's eight are all in or all out)
        if (in) mx4_load8<VEC>(x + src * ld + col, v);
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
        }
        uint32_t top = mx4_top8(v);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t s = mx4_scale_of(top);
        const float inv = mx4_inverse(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = s == 255u ? 0.f : v[i] * inv;
        if (in) *reinterpret_cast<uint32_t*>(codes + row * (long long)(k >> 1) + (col >> 1)) = mx4_encode8(v);
        // the four scales of 128 entries as one word
        uint32_t word = s << (8 * ((lane >> 2) & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if ((lane & 15) == 0)
            *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(scale_row, (long long)c * 8 + (lane >> 4) * 4, kg)) = word;
    }
}

// A stack of matrices: `rows` rows each, whose scales take rb * 128 scale rows.
template <typename T>
__global__ void __launch_bounds__(128)
mx4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, long long all_rows, int rows, int k, T* out) {
    pdl_wait();
    pdl_launch_dependents();
    const long long kg = mx4_atoms_k(k), rb = (rows + 127) / 128, per = k >> 3, n = all_rows * per;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long row = i / per, g = row / rows, r = row - g * rows;
        const int col = (int)(i - row * per) * 8;
        const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + i * 4);
        const uint32_t s = scales[(size_t)g * rb * kg * MX4_ATOM + mx4_scale_at(r, col >> 5, kg)];
        const float f = s == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(s ? s << 23 : 0x00400000u);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t c = (word >> (4 * j)) & 15u, e = (c >> 1) & 3u, m = c & 1u;
            // e2m1 as float32: 0.5 m for exponent 0, else 2^(e - 1) (1 + m / 2)
            const uint32_t bits = e ? ((e + 126u) << 23) | (m << 22) : (m ? 0x3f000000u : 0u);
            v[j] = __uint_as_float(bits | ((c & 8u) << 28)) * f;
        }
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(out + i * 8)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(out + i * 8)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                u[j] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(out + i * 8) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
}

template <typename T, bool VEC>
static int mx4_launch(const T* x, long long ld, int rows, int k, uint8_t* codes, uint8_t* scales, int pad_rows, const int* offsets,
                      const int* place, int E, int top_k, cudaStream_t stream) {
    const long long warps = (long long)pad_rows * ((k + MX4_CHUNK - 1) / MX4_CHUNK), blocks = (warps + 3) / 4;
    const long long most = 16ll * rllm_sm_count();
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    if (offsets)
        return rllm_launch(mx4_quantize_kernel<T, VEC, true>, grid, dim3(128), 0, stream, x, ld, rows, k, codes, scales, pad_rows,
                           offsets, place, E, top_k);
    return rllm_launch(mx4_quantize_kernel<T, VEC, false>, grid, dim3(128), 0, stream, x, ld, rows, k, codes, scales, pad_rows,
                       offsets, place, E, top_k);
}

// x [rows, k] with rows ld apart -> codes [rows, k / 2] (16-byte aligned), scales.  k a multiple of 32.  pad != 0: the scales of
// the rows behind the last one, up to a multiple of 128, are written too (zeros).  offsets int32 [E + 1] (sorted rows, see
// above): then `rows` is the number of sorted rows and `place`, if given, int32 [rows].
RLLM_API int rllm_mx4_quantize(const void* x, int dt, long long ld, int rows, int k, void* codes, void* scales, int pad,
                               const int* offsets, const int* place, int E, int top_k, cudaStream_t stream) {
    if (rows <= 0 || k <= 0) return 0;
    if ((k % MX4_BLOCK) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 15) || (offsets && (E <= 0 || pad)) || (place && top_k <= 0) ||
        (place && !offsets) || rows > 0x7fffff00)
        return (int)cudaErrorInvalidValue;
    const int pad_rows = pad ? (rows + 127) / 128 * 128 : rows;
    const int esize = dt == RLLM_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)x & 15) == 0 && (ld * esize) % 16 == 0;
#define MX4_Q(T, VEC) \
    return mx4_launch<T, VEC>((const T*)x, ld, rows, k, (uint8_t*)codes, (uint8_t*)scales, pad_rows, offsets, place, E, top_k, stream)
    if (dt == RLLM_F32) { if (vec) { MX4_Q(float, true); } MX4_Q(float, false); }
    if (vec) { MX4_Q(bf16, true); }
    MX4_Q(bf16, false);
#undef MX4_Q
}

// out [matrices * rows, k] contiguous, float32 or bfloat16, 16-byte aligned
RLLM_API int rllm_mx4_dequantize(const void* codes, const void* scales, long long matrices, int rows, int k, void* out, int dt,
                                 cudaStream_t stream) {
    if (matrices <= 0 || rows <= 0 || k <= 0) return 0;
    if ((k % MX4_BLOCK) || ((uintptr_t)codes & 3) || ((uintptr_t)out & 15)) return (int)cudaErrorInvalidValue;
    const long long blocks = (matrices * rows * (k / 8) + 127) / 128, most = 16ll * rllm_sm_count();
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    if (dt == RLLM_F32)
        return rllm_launch(mx4_dequantize_kernel<float>, grid, dim3(128), 0, stream, (const uint8_t*)codes, (const uint8_t*)scales,
                           matrices * rows, rows, k, (float*)out);
    return rllm_launch(mx4_dequantize_kernel<bf16>, grid, dim3(128), 0, stream, (const uint8_t*)codes, (const uint8_t*)scales,
                       matrices * rows, rows, k, (bf16*)out);
}

RLLM_PACKED(rllm_mx4_quantize)
RLLM_PACKED(rllm_mx4_dequantize)
