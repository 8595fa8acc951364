// Rows to microscaled 4-bit numbers and back (mx4.cuh has the format and its layout).
//
//   mx4_quantize    codes and scales of the rows of x [rows, k] (float32 or bfloat16, any row stride).  With `offsets` the rows are
//                   those of routed experts: x has a row per token (`place` given: pair p of token p / top_k goes to row
//                   place[p] of the sorted rows) or the sorted rows themselves, and the scales lie in the order of the products'
//                   row tiles: expert e's rows begin a new block of 128 scale rows, the one behind the blocks of the experts before it.
//   mx4_dequantize  the values that codes and scales stand for, exact in float32 and in bfloat16.
//
// Both read and write every byte once; a warp takes up to four runs of 256 neighbouring entries of a row (all their loads in flight at
// once), a lane eight entries of each, so that loads are 512 or 1,024 and code stores 128 contiguous bytes; the four lanes of a block
// find its largest magnitude with two shuffles.  2,047 x 12,288 bfloat16: 12.0 us to quantise (5.3 TB/s; with an address worked out for every run
// and eight maxima in place of three packed ones 15.4: it was bound by instructions), 11.8 us back (5.4 TB/s).
#include "mx4.cuh"

#define MQ_RUNS 4                            // runs of 256 entries of a warp

template <typename T> struct MqPart;
template <> struct MqPart<bf16> {
    uint4 u;
    template <bool VEC> __device__ __forceinline__ void load(const bf16* p) {
        if (VEC) { u = *reinterpret_cast<const uint4*>(p); return; }
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
        u = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
    }
    __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ uint32_t codes(int lane, uint32_t& word) const {
        float v[8];
        mx4_unpack(u, v);
        return mx4_quantize8(v, mx4_top8(u), lane, word);
    }
};
template <> struct MqPart<float> {
    float v8[8];
    template <bool VEC> __device__ __forceinline__ void load(const float* p) { mx4_load8<VEC>(p, v8); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) v8[i] = 0.f;
    }
    __device__ __forceinline__ uint32_t codes(int lane, uint32_t& word) const { return mx4_quantize8(v8, mx4_top8(v8), lane, word); }
};

template <typename T, bool VEC, bool SORTED>
__global__ void __launch_bounds__(128)
mx4_quantize_kernel(const T* x, long long ld, int rows, int k, uint8_t* codes, uint8_t* scales, unsigned n_warps, unsigned per_row,
                    const int* offsets, const int* place, int E, int top_k) {
    // the kernels behind may start once the ones before are complete: a product reads its weights ahead of its own wait, and
    // those may be what the kernel before this one wrote
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const unsigned w = blockIdx.x * 4u + (threadIdx.x >> 5);
    if (w >= n_warps) return;
    const unsigned item = w / per_row;
    const int chunks = (k + MX4_CHUNK - 1) / MX4_CHUNK, c0 = (int)(w - item * per_row) * MQ_RUNS;
    MqPart<T> part[MQ_RUNS];
    const bool here = SORTED || item < (unsigned)rows;           // (rows behind the last one get scales of zero)
    const int col0 = c0 * MX4_CHUNK + lane * 8, left = here ? k - col0 : 0;      // (k is a multiple of 32: a lane's eight are all in or all out)
    const T* from = x + item * ld + col0;
#pragma unroll
    for (int i = 0; i < MQ_RUNS; ++i) {
        if (i * MX4_CHUNK < left) part[i].template load<VEC>(from + i * MX4_CHUNK);
        else part[i].zero();
    }
    uint32_t code[MQ_RUNS], word[MQ_RUNS];
#pragma unroll
    for (int i = 0; i < MQ_RUNS; ++i) code[i] = part[i].codes(lane, word[i]);
    auto store = [&](long long row, long long scale_row) {
        uint8_t* code_to = codes + row * (long long)(k >> 1) + (col0 >> 1);
        uint8_t* scale_to = scales + mx4_scale_at(scale_row, (long long)c0 * 8 + (lane >> 4) * 4, 2ll * chunks);
#pragma unroll
        for (int i = 0; i < MQ_RUNS; ++i) {
            if (c0 + i >= chunks) break;
            if (i * MX4_CHUNK < left) *reinterpret_cast<uint32_t*>(code_to + i * (MX4_CHUNK / 2)) = code[i];
            if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(scale_to + i * 2 * MX4_ATOM) = word[i];
        }
    };
    if constexpr (!SORTED) store(item, item);
    else for (int j = 0; j < top_k; ++j) {                       // a token's row goes to the places of its pairs
        const int row = place ? place[(long long)item * top_k + j] : (int)item;
        if (row < 0 || row >= rows) continue;
        // the row's expert is the first that ends behind it; its rows begin behind the row tiles of the experts before
        int before = 0, tiles = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + lane, end = e < E ? offsets[e + 1] : 0x7fffffff;
            const unsigned past = __ballot_sync(0xffffffffu, end <= row);
            if (past == 0) break;
            before += __popc(past);
            tiles += __reduce_add_sync(0xffffffffu, end <= row ? (end - offsets[e] + 127) >> 7 : 0);
        }
        if (before >= E) continue;
        const long long scale_row = (long long)tiles * 128 + (row - offsets[before]);
        // (offsets that do not rise from 0 to the number of rows: nothing outside the scales is written)
        if (scale_row >= 0 && scale_row < ((long long)((rows + 127) >> 7) + E) * 128) store(row, scale_row);
    }
}

// A stack of matrices: `rows` rows each, whose scales take rb * 128 scale rows.
template <typename T>
__global__ void __launch_bounds__(128)
mx4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, unsigned rows, int k, T* out, unsigned n_warps, unsigned per_row) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const unsigned w = blockIdx.x * 4u + (threadIdx.x >> 5);
    if (w >= n_warps) return;
    const unsigned row = w / per_row, g = row / rows, r = row - g * rows;
    const int c0 = (int)(w - row * per_row) * MQ_RUNS;
    const long long kg = mx4_atoms_k(k), base = (long long)row * k;
    const uint8_t* sc = scales + (size_t)g * ((rows + 127) >> 7) * kg * MX4_ATOM;
    uint32_t word[MQ_RUNS], s[MQ_RUNS];
#pragma unroll
    for (int i = 0; i < MQ_RUNS; ++i) {
        const int col = (c0 + i) * MX4_CHUNK + lane * 8;
        word[i] = col < k ? *reinterpret_cast<const uint32_t*>(codes + ((base + col) >> 1)) : 0u;
        s[i] = col < k ? sc[mx4_scale_at(r, col >> 5, kg)] : 0u;
    }
#pragma unroll
    for (int i = 0; i < MQ_RUNS; ++i) {
        const int col = (c0 + i) * MX4_CHUNK + lane * 8;
        if (col >= k) break;
        const float f = s[i] == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(s[i] ? s[i] << 23 : 0x00400000u);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // the three bits of the magnitude as a float32's lowest exponent bits and highest mantissa bit: the number times 2^-126
            const uint32_t mag = (j <= 5 ? word[i] << (22 - 4 * j) : word[i] >> (4 * j - 22)) & 0x01c00000u;
            v[j] = __uint_as_float(mag | ((word[i] << (28 - 4 * j)) & 0x80000000u)) * 8.507059173023462e37f * f;
        }
        T* o = out + base + col;
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                u[j] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
}

// Warps for `rows` rows of k entries: how many a row takes, and all of them (0: more than one launch can have).
static unsigned mq_warps(long long rows, int k, unsigned& per_row) {
    per_row = (unsigned)((k + MX4_CHUNK * MQ_RUNS - 1) / (MX4_CHUNK * MQ_RUNS));
    const long long n = rows * per_row;
    return n < 0xfffffff0ll ? (unsigned)n : 0u;
}

// items: rows to read, with pad those whose scales are written
template <typename T, bool VEC>
static int mx4_launch(const T* x, long long ld, int rows, int k, uint8_t* codes, uint8_t* scales, int items, const int* offsets,
                      const int* place, int E, int top_k, cudaStream_t stream) {
    unsigned per_row;
    const unsigned n = mq_warps(items, k, per_row);
    if (!n) return (int)cudaErrorInvalidValue;
    const dim3 grid(n / 4 + (n % 4 != 0));
    if (offsets)
        return rllm_launch(mx4_quantize_kernel<T, VEC, true>, grid, dim3(128), 0, stream, x, ld, rows, k, codes, scales, n, per_row,
                           offsets, place, E, top_k);
    return rllm_launch(mx4_quantize_kernel<T, VEC, false>, grid, dim3(128), 0, stream, x, ld, rows, k, codes, scales, n, per_row,
                       offsets, place, E, top_k);
}

// x [rows, k] with rows ld apart -> codes [rows, k / 2] (16-byte aligned), scales.  k a multiple of 32.  pad != 0: the scales of
// the rows behind the last one, up to a multiple of 128, are written too (zeros).  offsets int32 [E + 1] (sorted rows, see
// above): then `rows` is the number of sorted rows and `place`, if given, int32 [rows].
RLLM_API int rllm_mx4_quantize(const void* x, void* codes, void* scales, const int* offsets, const int* place, long long ld, int dt,
                               int rows, int k, int pad, int E, int top_k, cudaStream_t stream) {
    if (rows <= 0 || k <= 0) return 0;
    if ((k % MX4_BLOCK) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 15) || (offsets && (E <= 0 || pad)) || (place && (top_k <= 0 || rows % top_k)) ||
        (place && !offsets) || rows > 0x7fffff00)
        return (int)cudaErrorInvalidValue;
    const int items = pad ? (rows + 127) / 128 * 128 : place ? rows / top_k : rows;
    const int esize = dt == RLLM_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)x & 15) == 0 && (ld * esize) % 16 == 0;
#define MX4_Q(T, VEC) \
    return mx4_launch<T, VEC>((const T*)x, ld, rows, k, (uint8_t*)codes, (uint8_t*)scales, items, offsets, place, E, place ? top_k : 1, stream)
    if (dt == RLLM_F32) { if (vec) { MX4_Q(float, true); } MX4_Q(float, false); }
    if (vec) { MX4_Q(bf16, true); }
    MX4_Q(bf16, false);
#undef MX4_Q
}

// out [matrices * rows, k] contiguous, float32 or bfloat16, 16-byte aligned
RLLM_API int rllm_mx4_dequantize(const void* codes, const void* scales, void* out, long long matrices, int rows, int k, int dt,
                                 cudaStream_t stream) {
    if (matrices <= 0 || rows <= 0 || k <= 0) return 0;
    unsigned per_row;
    const unsigned n = mq_warps(matrices * rows, k, per_row);
    if ((k % MX4_BLOCK) || ((uintptr_t)codes & 3) || ((uintptr_t)out & 15) || !n) return (int)cudaErrorInvalidValue;
    const dim3 grid(n / 4 + (n % 4 != 0));
    if (dt == RLLM_F32)
        return rllm_launch(mx4_dequantize_kernel<float>, grid, dim3(128), 0, stream, (const uint8_t*)codes, (const uint8_t*)scales,
                           (unsigned)rows, k, (float*)out, n, per_row);
    return rllm_launch(mx4_dequantize_kernel<bf16>, grid, dim3(128), 0, stream, (const uint8_t*)codes, (const uint8_t*)scales,
                       (unsigned)rows, k, (bf16*)out, n, per_row);
}

RLLM_PACKED(rllm_mx4_quantize)
RLLM_PACKED(rllm_mx4_dequantize)
