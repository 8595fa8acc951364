// Products of microscaled 4-bit numbers on the Blackwell tensor cores: C[r, n] = sum_k Qa[r, k] Qb[n, k] with both operands as codes
// and scales (mx4.cuh), tcgen05.mma of kind mxf4 (block scales of 32 along K), float32 accumulation in tensor memory.
//
// Many rows, and the rows of routed experts.  The machinery of gemm_group.cu: persistent CTAs walk over 128 x 256 tiles, a ring of stages filled
// by TMA, one thread that issues the products, every mbarrier wait bounded.  What differs:
//   * a stage holds 256 entries along K: rows of 128 bytes as in the bfloat16 kernels (so the same 128-byte swizzle and the same
//     descriptors), and beside them the scales, 1,024 bytes for 128 rows, which arrive by plain bulk copies in the order in which
//     tcgen05.cp.32x128b.warpx4 spreads them over tensor memory: four columns for 128 rows and 128 entries along K, of which the instruction's
//     scale id picks the two bytes of its 64 entries;
//   * every stage has tensor-memory columns of its own for its scales: they are overwritten only when the products that read them
//     have released the stage;
//   * the accumulator takes 256 of the 512 columns, so there is one: eight epilogue warps take it into registers (128 a thread) and hand it
//     back before they convert and store.
// The rows of A may be sorted by expert (offsets int32 [E + 1] on the device): expert e's rows form row tiles of their own, counted by
// every CTA itself, whose scales lie in the same order (rllm_mx4_quantize); its matrix is number e of the stack B.
// The gated product: B is a stack of gate and up matrices in turn; a tile holds 128 gate rows and the 128 up rows of the same index.
#include "mx4_tc.cuh"

// mx4.cu
RLLM_API int rllm_mx4_quantize(const void* x, void* codes, void* scales, const int* offsets, const int* place, long long ld, int dt,
                               int rows, int k, int pad, int E, int top_k, cudaStream_t stream);

#define GM_BM 128
#define GM_BN 256
#define GM_STAGES 4
#define GM_THREADS 320
#define GM_MAX_E 1024
#define GM_A_BYTES (GM_BM * 128)
#define GM_B_BYTES (GM_BN * 128)
#define GM_STAGE_BYTES (GM_A_BYTES + GM_B_BYTES + 3 * MX4_SF_BYTES)
#define GM_SF_COLS 32                                      // tensor-memory columns of a stage's scales: 8 of A, 16 of B

enum { GM_EPI_STORE = 0, GM_EPI_ACCUM = 1, GM_EPI_GATED = 2 };
enum { GM_ERR_FULL = 31, GM_ERR_EMPTY = 32, GM_ERR_ACC = 33 };

template <typename TC> __device__ __forceinline__ void gm_store32(TC* dst, const float (&v)[32], int n_valid) {
    if (n_valid >= 32 && ((uintptr_t)dst & 15) == 0) {
        if constexpr (sizeof(TC) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                reinterpret_cast<float4*>(dst)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t u[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[8 * j + 2 * q], v[8 * j + 2 * q + 1]);
                    u[q] = *reinterpret_cast<const uint32_t*>(&b);
                }
                reinterpret_cast<uint4*>(dst)[j] = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < n_valid) dst[j] = from_f<TC>(v[j]);
    }
}

// ---------------------------------------------------------------- the kernel
template <typename TC, int EPI>
__global__ void __launch_bounds__(GM_THREADS, 1)
gemm_mx4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const uint8_t* sfa, const uint8_t* sfb,
                TC* C, long long ldc, const int* offsets, int E, int rows, int N, int K, int ahead, const GluForm glu, int* err) {
    constexpr bool GATED = EPI == GM_EPI_GATED;
    constexpr int BN_OUT = GATED ? GM_BN / 2 : GM_BN;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t full_bar[GM_STAGES];
    __shared__ __align__(8) uint64_t empty_bar[GM_STAGES];
    __shared__ __align__(8) uint64_t acc_full, acc_empty;
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    __shared__ int s_row[GM_MAX_E + 1];              // an expert's first row
    __shared__ int s_tile[GM_MAX_E + 1];             // its first row tile

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nkb = (K + MX4_CHUNK - 1) / MX4_CHUNK, n_tiles = (N + BN_OUT - 1) / BN_OUT;
    const int rb_n = (N + 127) >> 7;                 // blocks of 128 scale rows of one matrix of B
    const size_t rb_bytes = (size_t)nkb * MX4_SF_BYTES;
    const int rb_most = offsets ? ((rows + GM_BM - 1) / GM_BM + E) : (rows + GM_BM - 1) / GM_BM;
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
        for (int s = 0; s < GM_STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        mbar_init(&acc_full, 1);
        mbar_init(&acc_empty, 256);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_slot, 512);
        tmem_relinquish();
    }
    if (offsets) pdl_wait();                          // rows and offsets are written by the kernels before
    if (warp == 2) {                                 // first rows and first row tiles of the experts, 32 at a time
        int run = 0;
        for (int e0 = 0; e0 <= E; e0 += 32) {
            const int e = e0 + lane;
            const int first = e > E ? 0 : offsets ? min(max(offsets[e], 0), rows) : (e == 0 ? 0 : rows);
            const int next = e >= E ? first : offsets ? min(max(offsets[e + 1], 0), rows) : rows;
            const int t = e < E ? (max(next - first, 0) + GM_BM - 1) / GM_BM : 0;
            int incl = t;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, m);
                if (lane >= m) incl += up;
            }
            if (e <= E) {
                s_row[e] = first;
                s_tile[e] = min(run + incl - t, rb_most);
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    const int m_tiles = s_tile[E], total_tiles = m_tiles * n_tiles;
    // tile -> its expert, row tile, first row, rows of the expert from there on, first column (row tiles fastest)
    auto place = [&](int tile, int& e, int& mt, int& m0, int& m_end, int& n0) {
        mt = tile % m_tiles;
        int lo = 0, hi = E;                          // the last expert whose first tile is <= mt (and that has tiles)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_tile[mid] <= mt) lo = mid; else hi = mid;
        }
        e = lo;
        m0 = s_row[lo] + (mt - s_tile[lo]) * GM_BM;
        m_end = s_row[lo + 1];
        n0 = tile / m_tiles * BN_OUT;
    };

    if (warp == 0 && lane == 0) {
        // ---- producer: one continuous ring over all of this CTA's tiles
        int it = 0, issued = 0;
        bool ok = true;
        auto load_b = [&](int s, int kb, int e, int n0) {
            unsigned char* b_s = smem + (size_t)s * GM_STAGE_BYTES + GM_A_BYTES;
            unsigned char* f_s = b_s + GM_B_BYTES + MX4_SF_BYTES;
            const int rb = n0 >> 7;
            if (GATED) {
                const long long g = 2ll * e;
                tma_load_2d(b_s, &tmB, kb * 128, (int)(g * N) + n0, &full_bar[s]);
                tma_load_2d(b_s + GM_B_BYTES / 2, &tmB, kb * 128, (int)((g + 1) * N) + n0, &full_bar[s]);
                bulk_load(f_s, sfb + (g * rb_n + rb) * rb_bytes + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
                bulk_load(f_s + MX4_SF_BYTES, sfb + ((g + 1) * rb_n + rb) * rb_bytes + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
            } else {
                // (the second 128 rows of a matrix's last tile may not exist: whatever comes in belongs to columns that are dropped)
                const long long r0 = (long long)e * rb_n;
                tma_load_2d(b_s, &tmB, kb * 128, e * N + n0, &full_bar[s]);
                tma_load_2d(b_s + GM_B_BYTES / 2, &tmB, kb * 128, e * N + n0 + 128, &full_bar[s]);
                bulk_load(f_s, sfb + (r0 + rb) * rb_bytes + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
                bulk_load(f_s + MX4_SF_BYTES, sfb + (r0 + min(rb + 1, rb_n - 1)) * rb_bytes + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES,
                          &full_bar[s]);
            }
        };
        // weights that are settled do not depend on the kernel before: the first stages' start ahead of the wait
        const int head = ahead && !offsets && blockIdx.x < total_tiles ? min(GM_STAGES, nkb) : 0;
        if (head) {
            int e, mt, m0, m_end, n0;
            place(blockIdx.x, e, mt, m0, m_end, n0);
            for (int s = 0; s < head; ++s) {
                mbar_expect_tx(&full_bar[s], GM_STAGE_BYTES);
                load_b(s, s, e, n0);
            }
        }
        if (!offsets) pdl_wait();
        for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x) {
            int e, mt, m0, m_end, n0;
            place(tile, e, mt, m0, m_end, n0);
            const uint8_t* sf_rows = sfa + (size_t)min(mt, rb_most - 1) * rb_bytes;
            for (int kb = 0; kb < nkb; ++kb, ++it) {
                const int s = it % GM_STAGES;
                const uint32_t ph = (it / GM_STAGES) & 1;
                if (!mbar_wait(&empty_bar[s], ph ^ 1, &abort_flag)) {
                    if (!abort_flag) { atomicExch(err, GM_ERR_EMPTY); abort_flag = 1; }
                    ok = false;
                    break;
                }
                unsigned char* a_s = smem + (size_t)s * GM_STAGE_BYTES;
                if (it >= head) mbar_expect_tx(&full_bar[s], GM_STAGE_BYTES);
                tma_load_2d(a_s, &tmA, kb * 128, m0, &full_bar[s]);
                bulk_load(a_s + GM_A_BYTES + GM_B_BYTES, sf_rows + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
                if (it >= head) load_b(s, kb, e, n0);
                issued = it + 1;
            }
        }
        if (abort_flag) {
            // copies already issued must land before the CTA's shared memory goes away
            volatile int no_abort = 0;
            for (int i = max(0, issued - GM_STAGES); i < issued; ++i)
                mbar_wait(&full_bar[i % GM_STAGES], (i / GM_STAGES) & 1, &no_abort);
        }
    } else if (warp == 1 && lane == 0) {
        // ---- issuer: the stage's scales to tensor memory, then four products of 64 entries along K
        int it = 0, local = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x, ++local) {
            if (!mbar_wait(&acc_empty, (local & 1) ^ 1, &abort_flag)) {
                if (!abort_flag) { atomicExch(err, GM_ERR_ACC); abort_flag = 1; }
                break;
            }
            tc_fence_after();
            for (int kb = 0; kb < nkb; ++kb, ++it) {
                const int s = it % GM_STAGES;
                const uint32_t ph = (it / GM_STAGES) & 1;
                if (!mbar_wait(&full_bar[s], ph, &abort_flag)) {
                    if (!abort_flag) { atomicExch(err, GM_ERR_FULL); abort_flag = 1; }
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t a_addr = s_addr(smem + (size_t)s * GM_STAGE_BYTES);
                const uint32_t f_addr = a_addr + GM_A_BYTES + GM_B_BYTES;
                const uint32_t t_a = tmem_base + GM_BN + s * GM_SF_COLS, t_b = t_a + 8;
#pragma unroll
                for (int g = 0; g < 2; ++g) {                // 128 entries along K each
                    tmem_cp_atom(t_a + 4 * g, smem_desc_atom(f_addr + g * MX4_ATOM));
                    tmem_cp_atom(t_b + 8 * g, smem_desc_atom(f_addr + MX4_SF_BYTES + g * MX4_ATOM));
                    tmem_cp_atom(t_b + 8 * g + 4, smem_desc_atom(f_addr + 2 * MX4_SF_BYTES + g * MX4_ATOM));
                }
                const uint64_t a_desc = smem_desc_sw128(a_addr), b_desc = smem_desc_sw128(a_addr + GM_A_BYTES);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)               // 64 entries = 32 bytes along K: +2 in 16-byte units
                    umma_mxf4(tmem_base, a_desc + 2 * kk, b_desc + 2 * kk, idesc_mxf4(GM_BM, GM_BN, (kk & 1) * 2), t_a + 4 * (kk >> 1),
                              t_b + 8 * (kk >> 1), (kb | kk) != 0);
                umma_commit(&empty_bar[s]);
            }
            if (ok) umma_commit(&acc_full);
        }
    } else if (warp >= 2) {
        // ---- epilogue: warp w may touch the lanes 32 * (w % 4) .. + 31; the first four take the first half of the columns
        if (!offsets) pdl_wait();
        const int quarter = warp & 3, half = (warp - 2) >> 2, row = quarter * 32 + lane;
        int local = 0;
        for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++local) {
            int e, mt, m0, m_end, n0;
            place(tile, e, mt, m0, m_end, n0);
            const int gm = m0 + row;
            bool ok = mbar_wait(&acc_full, local & 1, &abort_flag);
            if (!ok && !abort_flag) { atomicExch(err, GM_ERR_ACC); abort_flag = 1; }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16);
            uint32_t r[4][32];
            if (GATED) {
                tmem_ld32(taddr + half * 64, r[0]);
                tmem_ld32(taddr + half * 64 + 32, r[1]);
                tmem_ld32(taddr + 128 + half * 64, r[2]);
                tmem_ld32(taddr + 128 + half * 64 + 32, r[3]);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_ld32(taddr + half * 128 + q * 32, r[q]);
            }
            tmem_ld_wait();
            tc_fence_before();
            mbar_arrive(&acc_empty);
            if (gm < m_end) {
#pragma unroll
                for (int q = 0; q < (GATED ? 2 : 4); ++q) {
                    const int gn = n0 + (GATED ? half * 64 : half * 128) + q * 32;
                    if (gn >= N) break;
                    TC* dst = C + (size_t)gm * ldc + gn;
                    const int n_valid = min(32, N - gn);
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        v[j] = GATED ? glu_apply(glu, __uint_as_float(r[q][j]), __uint_as_float(r[GATED ? q + 2 : q][j])) : __uint_as_float(r[q][j]);
                    if (EPI == GM_EPI_ACCUM) {
                        if (sizeof(TC) == 4 && n_valid >= 32 && ((uintptr_t)dst & 15) == 0) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float4 c4 = reinterpret_cast<const float4*>(dst)[j];
                                v[4 * j] += c4.x; v[4 * j + 1] += c4.y; v[4 * j + 2] += c4.z; v[4 * j + 3] += c4.w;
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) if (j < n_valid) v[j] += to_f<TC>(dst[j]);
                        }
                    }
                    gm_store32<TC>(dst, v, n_valid);
                }
            }
        }
        pdl_launch_dependents();
    }
    __syncwarp();          // the lanes that had no role meet the elected one: the barrier below wants whole warps
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// ---------------------------------------------------------------- host side
// A: codes [rows, K / 2] and scales; B: codes [matrices * N, K / 2] and the matrices' scales one after another (matrices: E, gated
// 2 E, gate and up in turn).  K a multiple of 32, all bases 16-byte aligned.  offsets int32 [E + 1] on the device (null: E is 1, all
// rows are its).  epilogue 0 store, 1 add into a float32 C, 2 gated (GluForm).  ahead: B is settled and may be read before the
// kernels before have ended.  Returns 0, a cudaError_t or 30000 + CUresult of the tensor-map encoder.
static int rllm_gemm_mx4(const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales, void* C, int c_dtype,
                           long long ldc, const int* offsets, int E, int rows, int N, int K, int epilogue, int ahead, float glu_limit,
                           float glu_alpha, float glu_shift, int* err, cudaStream_t stream) {
    if (rows <= 0 || N <= 0) return 0;
    const long long matrices = (long long)E * (epilogue == GM_EPI_GATED ? 2 : 1);
    if (E <= 0 || E > GM_MAX_E || (!offsets && E != 1) || K <= 0 || (K % MX4_BLOCK) || !err || ldc < N || matrices * N > 0x7fffff00LL ||
        rows > 0x7fffff00 || ((uintptr_t)a_codes & 15) || ((uintptr_t)a_scales & 15) || ((uintptr_t)b_codes & 15) ||
        ((uintptr_t)b_scales & 15) || (epilogue == GM_EPI_ACCUM && c_dtype != RLLM_F32))
        return (int)cudaErrorInvalidValue;
    CUtensorMap ta, tb;
    int st = mx4_tmap(&ta, a_codes, rows, K, GM_BM);
    if (st) return st;
    st = mx4_tmap(&tb, b_codes, matrices * N, K, 128);
    if (st) return st;
    const GluForm glu = GluForm{glu_limit, glu_alpha, glu_shift};
    const int bn_out = epilogue == GM_EPI_GATED ? GM_BN / 2 : GM_BN;
    const long long most = ((long long)(rows + GM_BM - 1) / GM_BM + (offsets ? E : 0)) * ((N + bn_out - 1) / bn_out);
    if (most > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    const int n_sm = rllm_sm_count(), grid = (int)(most < n_sm ? most : n_sm);
    constexpr int smem = GM_STAGES * GM_STAGE_BYTES + 1024;
    auto run = [&](auto kern, auto* out) -> int {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
        return rllm_launch(kern, dim3(grid), dim3(GM_THREADS), smem, stream, ta, tb, (const uint8_t*)a_scales, (const uint8_t*)b_scales,
                           out, ldc, offsets, E, rows, N, K, ahead, glu, err);
    };
    if (epilogue == GM_EPI_ACCUM) return run(gemm_mx4_kernel<float, GM_EPI_ACCUM>, (float*)C);
    if (epilogue == GM_EPI_GATED)
        return c_dtype == RLLM_F32 ? run(gemm_mx4_kernel<float, GM_EPI_GATED>, (float*)C) : run(gemm_mx4_kernel<bf16, GM_EPI_GATED>, (bf16*)C);
    if (epilogue == GM_EPI_STORE)
        return c_dtype == RLLM_F32 ? run(gemm_mx4_kernel<float, GM_EPI_STORE>, (float*)C) : run(gemm_mx4_kernel<bf16, GM_EPI_STORE>, (bf16*)C);
    return (int)cudaErrorInvalidValue;
}

TC_DEFINE_WAIT_CONTROLS(rllm_gemm_mx4)

// The whole product from rows x [rows of x, K] (float32 or bfloat16, ldx apart): they are quantised into `work` (codes, and from the next multiple
// of 1,024 bytes the scales), which rllm_gemm_mx4 then reads.  offsets, place, E, top_k as for rllm_mx4_quantize; `rows` sorted rows.
RLLM_API int rllm_mx4_product(const void* x, const int* offsets, const int* place, const void* w_codes, const void* w_scales, void* C,
                              void* work, int* err, long long ldx, long long ldc, int x_dtype, int c_dtype, int rows, int N, int K, int E,
                              int top_k, int epilogue, int ahead, float glu_limit, float glu_alpha, float glu_shift, cudaStream_t stream) {
    if (rows <= 0 || N <= 0) return 0;
    unsigned char* scales = (unsigned char*)work + (((size_t)rows * (size_t)(K / 2) + 1023) & ~(size_t)1023);
    const int st = rllm_mx4_quantize(x, work, scales, offsets, place, ldx, x_dtype, rows, K, 0, E, top_k, stream);
    if (st) return st;
    return rllm_gemm_mx4(work, scales, w_codes, w_scales, C, c_dtype, ldc, offsets, E, rows, N, K, epilogue, ahead, glu_limit, glu_alpha,
                         glu_shift, err, stream);
}

RLLM_PACKED(rllm_mx4_product)
