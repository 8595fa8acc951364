// Products of microscaled 4-bit numbers for few rows (decode): C[b, n] = sum_k Q(X)[b, k] W[n, k], at most 64 rows X [m, K] in bfloat16 or
// float32, W as codes and scales (mx4.cuh).  What it cannot do without is reading W once, 17 bytes for 32 entries; so W is the
// streamed M side (128 rows a CTA), the rows are the N side (16, 32 or 64 columns of the accumulator), and
//   * the rows become 4-bit numbers here: four warps read the CTA's part of X, quantise it and write it into the stage that the
//     product reads (the 128-byte swizzle and the scale atoms by hand), so that a product is one launch.  Every CTA repeats that for its part of K; at
//     up to 64 rows it is a fraction of the weights' time, and loads run several rows ahead;
//   * weights that are settled start ahead of the dependency wait, as in the bfloat16 kernels;
//   * a thread-block cluster of 2, 4 or 8 CTAs shares a tile's K where there are few tiles: partial sums are parked in shared memory, every CTA
//     adds and writes its share of the tile's rows, in rank order, which is ascending k (no atomics, no global scratch).  The number of
//     CTAs depends on W's shape alone, so a row's bits do not depend on the rows around it.
// The gated product: a CTA takes 128 gate rows and the 128 up rows of the same index, with an accumulator each.
#include "mx4_tc.cuh"

#define GR_THREADS 192

enum { GR_EPI_STORE = 0, GR_EPI_ACCUM = 1, GR_EPI_GATED = 2 };
enum { GR_ERR_FULL = 34, GR_ERR_EMPTY = 35, GR_ERR_ACC = 36 };

// what a lane holds of a row's 256 entries: eight, as they came
template <typename TX> struct RowPart;
template <> struct RowPart<bf16> {
    uint4 u;
    __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&v)[8]) const { mx4_unpack(u, v); }
};
template <> struct RowPart<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};

template <int BN, int STAGES, int EPI, typename TC, typename TX>
__global__ void __launch_bounds__(GR_THREADS, 1)
gemm_mx4_rows_kernel(const __grid_constant__ CUtensorMap tmW, const uint8_t* sfw, const TX* X, long long ldx, TC* C, long long ldc,
                     int m, int n, int K, int ahead, const GluForm glu, int* err) {
    constexpr bool GATED = EPI == GR_EPI_GATED;
    constexpr int WT = GATED ? 2 : 1;                        // tiles of 128 weight rows of a CTA
    constexpr int W_BYTES = 128 * 128, X_BYTES = BN * 128;
    constexpr int TX_BYTES = WT * (W_BYTES + MX4_SF_BYTES);  // what arrives by TMA and bulk copies
    constexpr int STAGE_BYTES = TX_BYTES + X_BYTES + MX4_SF_BYTES;
    constexpr int SF_COLS = WT * 8 + 8;                      // tensor-memory columns of a stage's scales
    constexpr int TMEM_COLS = WT * BN + STAGES * SF_COLS <= 128 ? 128 : WT * BN + STAGES * SF_COLS <= 256 ? 256 : 512;
    constexpr int U = sizeof(TX) == 2 ? 8 : 4;               // rows a warp has in flight
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t full_bar[STAGES];
    __shared__ __align__(8) uint64_t empty_bar[STAGES];
    __shared__ __align__(8) uint64_t acc_bar;
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    float* red = reinterpret_cast<float*>(smem);             // parked sums [weight tile][batch row][weight row]: the stages are free by then

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.y, n_splits = gridDim.y, n0 = blockIdx.x * 128;
    const int nkb = (K + MX4_CHUNK - 1) / MX4_CHUNK;
    const int kb0 = (int)((long long)nkb * split / n_splits), my_kb = (int)((long long)nkb * (split + 1) / n_splits) - kb0;
    const size_t rb_bytes = (size_t)nkb * MX4_SF_BYTES;
    const int x_warps = min(m, 4);                           // warps that have rows to quantise

    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmW) : "memory");
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1 + x_warps); mbar_init(&empty_bar[s], 1); }
        mbar_init(&acc_bar, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_slot, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    float v[WT][BN];                                         // the epilogue threads' accumulator rows
    bool ep_ok = true;

    if (warp == 0 && lane == 0) {
        // ---- the weights and their scales
        if (!ahead) pdl_wait();
        int issued = 0;
        const int rb_n = (n + 127) >> 7;
        for (int i = 0; i < my_kb; ++i) {
            const int kb = kb0 + i, s = i % STAGES;
            if (!mbar_wait(&empty_bar[s], ((i / STAGES) & 1) ^ 1, &abort_flag)) {
                if (!abort_flag) { atomicExch(err, GR_ERR_EMPTY); abort_flag = 1; }
                break;
            }
            unsigned char* w_s = smem + (size_t)s * STAGE_BYTES;
            mbar_expect_tx(&full_bar[s], TX_BYTES);
#pragma unroll
            for (int t = 0; t < WT; ++t) {
                tma_load_2d(w_s + t * W_BYTES, &tmW, kb * 128, t * n + n0, &full_bar[s]);
                bulk_load(w_s + WT * W_BYTES + X_BYTES + t * MX4_SF_BYTES,
                          sfw + ((size_t)t * rb_n + blockIdx.x) * rb_bytes + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
            }
            issued = i + 1;
        }
        if (ahead) pdl_wait();
        if (abort_flag) {
            // the copies already issued must land before the CTA's shared memory goes away; their barriers cannot complete any
            // more (the other arrivals may be missing), so every stage that is not full gets them from here
            volatile int no_abort = 0;
            for (int i = max(0, issued - STAGES); i < issued; ++i) {
                for (int a = 0; a < x_warps; ++a) mbar_arrive(&full_bar[i % STAGES]);
                mbar_wait(&full_bar[i % STAGES], (i / STAGES) & 1, &no_abort);
            }
        }
    } else if (warp == 1 && lane == 0) {
        // ---- issuer
        bool ok = true;
        for (int i = 0; i < my_kb; ++i) {
            const int s = i % STAGES;
            if (!mbar_wait(&full_bar[s], (i / STAGES) & 1, &abort_flag)) {
                if (!abort_flag) { atomicExch(err, GR_ERR_FULL); abort_flag = 1; }
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t w_addr = s_addr(smem + (size_t)s * STAGE_BYTES), x_addr = w_addr + WT * W_BYTES, f_addr = x_addr + X_BYTES;
            const uint32_t t_x = tmem_base + WT * BN + s * SF_COLS, t_w = t_x + 8;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                tmem_cp_atom(t_x + 4 * g, smem_desc_atom(f_addr + WT * MX4_SF_BYTES + g * MX4_ATOM));
#pragma unroll
                for (int t = 0; t < WT; ++t) tmem_cp_atom(t_w + t * 8 + 4 * g, smem_desc_atom(f_addr + t * MX4_SF_BYTES + g * MX4_ATOM));
            }
            const uint64_t x_desc = smem_desc_sw128(x_addr);
#pragma unroll
            for (int t = 0; t < WT; ++t) {
                const uint64_t w_desc = smem_desc_sw128(w_addr + t * W_BYTES);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    umma_mxf4(tmem_base + t * BN, w_desc + 2 * kk, x_desc + 2 * kk, idesc_mxf4(128, BN, (kk & 1) * 2),
                              t_w + t * 8 + 4 * (kk >> 1), t_x + 4 * (kk >> 1), (i | kk) != 0);
            }
            umma_commit(&empty_bar[s]);
        }
        if (ok) umma_commit(&acc_bar);
    } else if (warp >= 2) {
        // ---- first the rows of X into the stages: warp q takes rows q, q + 4, ...; stage by stage, U rows in flight
        pdl_wait();
        const int q = warp & 3;
        if (q < m) {
            const int per = (m - q + 3) >> 2, items = my_kb * per;      // item: stage item / per, row q + 4 (item % per)
            RowPart<TX> part[U];
            auto fetch = [&](RowPart<TX>& p, int item) {
                const int i = item / per, col = (kb0 + i) * MX4_CHUNK + lane * 8;
                if (item < items && col < K) p.load(X + (size_t)(q + 4 * (item - i * per)) * ldx + col);
                else p.zero();
            };
#pragma unroll
            for (int u = 0; u < U; ++u) fetch(part[u], u);
            bool ok = true;
            for (int base = 0; base < items && ok; base += U) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int item = base + u;
                    if (item < items && ok) {
                        const int i = item / per, r = q + 4 * (item - i * per), s = i % STAGES;
                        if (item == i * per && !mbar_wait(&empty_bar[s], ((i / STAGES) & 1) ^ 1, &abort_flag)) {
                            if (!abort_flag) { atomicExch(err, GR_ERR_EMPTY); abort_flag = 1; }
                            ok = false;
                        }
                        ok = __all_sync(0xffffffffu, ok);
                        if (ok) {
                            float f[8];
                            part[u].get(f);
                            uint32_t word;
                            const uint32_t code = mx4_quantize8(f, lane, word);
                            unsigned char* x_s = smem + (size_t)s * STAGE_BYTES + WT * W_BYTES;
                            *reinterpret_cast<uint32_t*>(x_s + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2))) = code;
                            if ((lane & 15) == 0)
                                *reinterpret_cast<uint32_t*>(x_s + X_BYTES + WT * MX4_SF_BYTES + (lane >> 4) * MX4_ATOM + (r & 31) * 16 +
                                                             (r >> 5) * 4) = word;
                            if (item == i * per + per - 1) {           // the warp's part of the stage is written
                                fence_async_smem();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(&full_bar[s]);
                            }
                        }
                    }
                    fetch(part[u], base + U + u);
                }
            }
        }
        // ---- then the accumulators (thread = weight row, registers = rows of X)
        const int row = q * 32 + lane;
#pragma unroll
        for (int t = 0; t < WT; ++t)
#pragma unroll
            for (int b = 0; b < BN; ++b) v[t][b] = 0.f;
        if (my_kb > 0) {
            ep_ok = mbar_wait(&acc_bar, 0, &abort_flag);
            if (!ep_ok && !abort_flag) { atomicExch(err, GR_ERR_ACC); abort_flag = 1; }
        }
        ep_ok = __all_sync(0xffffffffu, ep_ok);
        pdl_launch_dependents();
        if (ep_ok && my_kb > 0) {
            tc_fence_after();
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
#pragma unroll
            for (int t = 0; t < WT; ++t)
#pragma unroll
                for (int c0 = 0; c0 < BN; c0 += 16) tmem_ld16(taddr + t * BN + c0, v[t] + c0);
            tmem_ld_wait();
        }
        if (n_splits > 1) {
#pragma unroll
            for (int t = 0; t < WT; ++t)
#pragma unroll
                for (int b = 0; b < BN; ++b)
                    if (b < m) red[(t * BN + b) * 128 + row] = v[t][b];
        }
    }
    __syncwarp();          // the lanes that had no role meet the elected one: the barriers below want whole warps
    tc_fence_before();
    __syncthreads();
    // NB rows of X at a column of C, from b0 in steps of `step`: the old values are all on their way before the first is used
    constexpr int NB = 8;
    auto write = [&](int b0, int step, int col, const float (&sum)[WT][NB]) {
        if (col >= n || !ep_ok) return;
        TC* dst = C + (size_t)b0 * ldc + col;
        float old[NB];
        if (EPI == GR_EPI_ACCUM) {
#pragma unroll
            for (int i = 0; i < NB; ++i) old[i] = b0 + i * step < m ? to_f<TC>(dst[(size_t)(i * step) * ldc]) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            float o = GATED ? glu_apply(glu, sum[0][i], sum[WT - 1][i]) : sum[0][i];
            if (EPI == GR_EPI_ACCUM) o += old[i];
            if (b0 + i * step < m) dst[(size_t)(i * step) * ldc] = from_f<TC>(o);
        }
    };
    if (n_splits > 1) {
        // every thread of every CTA of the cluster comes here, whatever happened before.  #1: all sums are parked
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (warp >= 2) {
            // this CTA's 128 / n_splits weight rows; n_splits groups of threads take every n_splits-th row of X
            const int t = tid - 64, share = 128 / n_splits, row = split * share + (t & (share - 1));
            for (int b0 = t / share; b0 < m; b0 += NB * n_splits) {
                float sum[WT][NB];
                for (int z = 0; z < n_splits; ++z) {             // in rank order: ascending k
                    float f[WT][NB];
#pragma unroll
                    for (int w = 0; w < WT; ++w) {
                        uint32_t remote;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(s_addr(red + w * BN * 128 + row)), "r"(z));
#pragma unroll
                        for (int i = 0; i < NB; ++i) {
                            const int b = b0 + i * n_splits;
                            f[w][i] = 0.f;
                            if (b < m) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[w][i]) : "r"(remote + (uint32_t)b * 512u) : "memory");
                        }
                    }
#pragma unroll
                    for (int w = 0; w < WT; ++w)
#pragma unroll
                        for (int i = 0; i < NB; ++i) sum[w][i] = z ? sum[w][i] + f[w][i] : f[w][i];
                }
                write(b0, n_splits, n0 + row, sum);
            }
        }
        // #2: nobody reads another CTA's shared memory any more
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else if (warp >= 2) {
        const int row = (warp & 3) * 32 + lane;
#pragma unroll
        for (int b0 = 0; b0 < BN; b0 += NB) {
            float sum[WT][NB];
#pragma unroll
            for (int w = 0; w < WT; ++w)
#pragma unroll
                for (int i = 0; i < NB; ++i) sum[w][i] = v[w][b0 + i];
            if (b0 < m) write(b0, 1, n0 + row, sum);
        }
    }
    if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

// ---------------------------------------------------------------- host side
template <int BN, int STAGES, int EPI, typename TC, typename TX>
static int gr_launch(const CUtensorMap& tw, const void* sfw, const void* X, long long ldx, void* C, long long ldc, int m, int n, int K,
                     int ahead, const GluForm glu, int splits, int* err, cudaStream_t stream) {
    constexpr int WT = EPI == GR_EPI_GATED ? 2 : 1;
    constexpr int smem = STAGES * (WT * (128 * 128 + MX4_SF_BYTES) + BN * 128 + MX4_SF_BYTES) + 1024;
    static_assert(WT * BN * 128 * 4 <= STAGES * (WT * (128 * 128 + MX4_SF_BYTES) + BN * 128 + MX4_SF_BYTES), "parked sums fit the stages");
    auto kern = gemm_mx4_rows_kernel<BN, STAGES, EPI, TC, TX>;
    static bool attr_set = false;
    if (!attr_set) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
        attr_set = true;
    }
    return rllm_launch_cluster(kern, dim3((n + 127) / 128, splits), dim3(GR_THREADS), smem, stream, splits, tw, (const uint8_t*)sfw,
                               (const TX*)X, ldx, (TC*)C, ldc, m, n, K, ahead, glu, err);
}

// X [m, K] (m <= 64, rows ldx apart, 16-byte aligned rows) in float32 or bfloat16; W: codes [n, K / 2] and scales, gated: gate and up
// matrix of n rows each.  splits: 1, 2, 4 or 8 CTAs share a tile's K.  The rest as rllm_gemm_mx4.
RLLM_API int rllm_gemm_mx4_rows(const void* X, const void* w_codes, const void* w_scales, void* C, int* err, long long ldx, long long ldc,
                                int x_dtype, int c_dtype, int m, int n, int K, int epilogue, int splits, int ahead, float glu_limit,
                                float glu_alpha, float glu_shift, cudaStream_t stream) {
    if (m <= 0 || n <= 0) return 0;
    const bool gated = epilogue == GR_EPI_GATED;
    if (m > 64 || K <= 0 || (K % MX4_BLOCK) || !err || ldc < n || (long long)n > 0x3fffff00LL || ((uintptr_t)w_codes & 15) ||
        ((uintptr_t)w_scales & 15) || ((uintptr_t)X & 15) || ((ldx * (x_dtype == RLLM_F32 ? 4 : 2)) & 15) ||
        (splits != 1 && splits != 2 && splits != 4 && splits != 8) || (epilogue == GR_EPI_ACCUM && c_dtype != RLLM_F32))
        return (int)cudaErrorInvalidValue;
    CUtensorMap tw;
    const int st = mx4_tmap(&tw, w_codes, (long long)n * (gated ? 2 : 1), K, 128);
    if (st) return st;
    const GluForm glu = GluForm{glu_limit, glu_alpha, glu_shift};
#define GR_GO(BN, ST, EPI, TC, TX) return gr_launch<BN, ST, EPI, TC, TX>(tw, w_scales, X, ldx, C, ldc, m, n, K, ahead, glu, splits, err, stream)
#define GR_X(BN, ST, EPI, TC) { if (x_dtype == RLLM_F32) { GR_GO(BN, ST, EPI, TC, float); } GR_GO(BN, ST, EPI, TC, bf16); }
#define GR_BN(ST1, EPI, TC) { if (m <= 16) GR_X(16, ST1, EPI, TC) if (m <= 32) GR_X(32, ST1, EPI, TC) GR_X(64, ST1, EPI, TC) }
    if (epilogue == GR_EPI_STORE) { if (c_dtype == RLLM_F32) GR_BN(4, GR_EPI_STORE, float) GR_BN(4, GR_EPI_STORE, bf16) }
    if (epilogue == GR_EPI_ACCUM) GR_BN(4, GR_EPI_ACCUM, float)
    if (gated) { if (c_dtype == RLLM_F32) GR_BN(4, GR_EPI_GATED, float) GR_BN(4, GR_EPI_GATED, bf16) }
#undef GR_BN
#undef GR_X
#undef GR_GO
    return (int)cudaErrorInvalidValue;
}

TC_DEFINE_WAIT_CONTROLS(rllm_gemm_mx4_rows)

RLLM_PACKED(rllm_gemm_mx4_rows)
