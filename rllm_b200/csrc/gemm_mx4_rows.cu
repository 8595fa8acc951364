// Products of microscaled 4-bit numbers for few rows (decode): C[b, n] = sum_k Q(X)[b, k] W[n, k], rows X in bfloat16 or float32, W as
// codes and scales (mx4.cuh).  What it cannot do without is reading W once, 17 bytes for 32 entries; so W is the streamed M side (128 rows
// a CTA), 16, 32, 64 or 128 rows of X are the N side, the columns of the accumulator, and
//   * the rows become 4-bit numbers here: four warps read the CTA's part of X, quantise it and write it into the stage that the
//     product reads (the 128-byte swizzle and the scale atoms by hand), so that a product is one launch.  Every CTA repeats that for its part
//     of K.  It is latency that counts: no division in the loop, loads up to eight rows ahead, several rows side by side.  That is for up to
//     16 rows; more of them (TX uint8_t) come as codes and scales that a launch before has made, by the same copies as the weights;
//   * weights that are settled start ahead of the dependency wait, as in the bfloat16 kernels;
//   * a thread-block cluster of 2, 4 or 8 CTAs shares a tile's K where there are few tiles: partial sums are parked in shared memory, every
//     CTA adds and writes its share of the tile's rows, in rank order, which is ascending k (no atomics, no global scratch).  With the same
//     kernel and the same number of CTAs a row's bits do not depend on the rows around it.  But both follow from all the sizes, the number of
//     rows among them (ops.mx4_few_rows, mx4_row_splits): from one number of rows to another its sums may differ in their last bits;
//   * of a gated product the cluster's first half of CTAs takes 128 gate rows, the other half the 128 up rows of the same index.
// Gated 8 x 2 x 12,288 x 4,096: 12.4 us (53.5 MB, 4.3 TB/s); 1 x 4,096 x 4,096: 6.3 us for 8.9 MB, a chain of latencies: rows in, quantised, product, sums
// through the cluster, out; 1 x 151,936 x 4,096: 52 us (6.3 TB/s).
// With `offsets` (int32 [E + 1] on the device) the rows are those of routed experts, sorted: every expert's rows form chunks of BN, found by
// every CTA itself from blockIdx.z; a CTA without a chunk leaves at once.  X then holds the sorted rows, or the tokens' rows with `place`:
// row place[p] of the sorted ones is X's row p / top_k.
#include "mx4_tc.cuh"

enum { GR_EPI_STORE = 0, GR_EPI_ACCUM = 1, GR_EPI_GATED = 2 };
enum { GR_ERR_FULL = 34, GR_ERR_EMPTY = 35, GR_ERR_ACC = 36 };

struct GrSorted {
    const int *offsets, *place;
    int E, top_k, rows;
};

// what a lane holds of a row's 256 entries: eight, as they came
template <typename TX> struct RowPart;
template <> struct RowPart<uint8_t> {};
template <> struct RowPart<bf16> {
    uint4 u;
    __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ uint32_t codes(int lane, uint32_t& word) const {
        float v[8];
        mx4_unpack(u, v);
        return mx4_quantize8(v, mx4_top8(u), lane, word);
    }
};
template <> struct RowPart<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ uint32_t codes(int lane, uint32_t& word) const {
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        return mx4_quantize8(v, mx4_top8(v), lane, word);
    }
};

// QW: warps that quantise, CTAS: CTAs that an SM is to hold
template <int BN, int STAGES, int QW, int CTAS, int EPI, typename TC, typename TX>
__global__ void __launch_bounds__(64 + 32 * QW, CTAS)
gemm_mx4_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const uint8_t* sfw, const TX* X,
                     long long ldx, TC* C, long long ldc,
                     int m_all, int n, int K, int ahead, const GluForm glu, const GrSorted so, int* err) {
    constexpr bool GATED = EPI == GR_EPI_GATED;
    constexpr int HALVES = GATED ? 2 : 1;
    constexpr int W_BYTES = 128 * 128, X_BYTES = BN * 128;
    constexpr bool CODES = sizeof(TX) == 1;                  // X is the rows' scales, tmX their codes
    constexpr int STAGE_BYTES = W_BYTES + X_BYTES + 2 * MX4_SF_BYTES;        // weights, rows, scales of the weights, scales of the rows
    constexpr int TX_BYTES = CODES ? STAGE_BYTES : W_BYTES + MX4_SF_BYTES;   // what arrives by TMA and bulk copies
    constexpr int SF_COLS = 16;                              // tensor-memory columns of a stage's scales
    constexpr int TMEM_COLS = BN + STAGES * SF_COLS <= 128 ? 128 : 256;
    constexpr int THREADS = 64 + 32 * QW;
    constexpr int RPW = BN / QW;                             // rows a warp takes of a stage, at most
    constexpr int AHEAD = sizeof(TX) == 4 ? 4 : 8;           // rows it has in flight
    constexpr int DEPTH = AHEAD > RPW ? AHEAD / RPW : 1;     // stages that it reads ahead
    constexpr int COLS = BN * 4 / QW;                        // accumulator columns of an epilogue thread
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t full_bar[STAGES];       // the weights and their scales have arrived
    __shared__ __align__(8) uint64_t rows_bar[STAGES];       // the rows are written
    __shared__ __align__(8) uint64_t empty_bar[STAGES];
    __shared__ __align__(8) uint64_t acc_bar;
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    __shared__ int s_src[BN];
    float* red = reinterpret_cast<float*>(smem);             // parked sums [row of X][weight row]: the stages are free by then

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int ranks = gridDim.y, n_splits = ranks / HALVES, half = (int)blockIdx.y / n_splits, split = (int)blockIdx.y - half * n_splits;
    const int n0 = blockIdx.x * 128;
    const int nkb = (K + MX4_CHUNK - 1) / MX4_CHUNK;
    const int kb0 = (int)((long long)nkb * split / n_splits), my_kb = (int)((long long)nkb * (split + 1) / n_splits) - kb0;
    const size_t rb_bytes = (size_t)nkb * MX4_SF_BYTES;

    // the chunk of rows: the expert, the first row, how many
    int e = 0, r0 = (int)blockIdx.z * BN, m = min(BN, m_all - r0);
    if (so.offsets) {
        pdl_wait();                                          // the rows and their order are written by the kernels before
        int run = 0;
        m = 0;
        for (int e0 = 0; e0 < so.E && m == 0; e0 += 32) {
            const int me = e0 + lane;
            const int first = me < so.E ? min(max(so.offsets[me], 0), so.rows) : 0, end = me < so.E ? min(max(so.offsets[me + 1], 0), so.rows) : 0;
            const int c = (max(end - first, 0) + BN - 1) / BN;
            int incl = c;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += up;
            }
            const int z = (int)blockIdx.z - run;
            const unsigned hit = __ballot_sync(0xffffffffu, z < incl && z >= incl - c);
            if (hit) {
                const int at = __ffs(hit) - 1, before = __shfl_sync(0xffffffffu, incl - c, at);
                e = e0 + at;
                r0 = __shfl_sync(0xffffffffu, first, at) + (z - before) * BN;
                m = min(BN, __shfl_sync(0xffffffffu, end, at) - r0);
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (m <= 0) return;                                  // (the whole cluster: it has one blockIdx.z)
        if (so.place) {
            for (int i = tid; i < BN; i += THREADS) s_src[i] = 0;
            __syncthreads();
            for (int p = tid; p < so.rows; p += THREADS) {
                const int r = so.place[p] - r0;
                if (r >= 0 && r < m) s_src[r] = p / so.top_k;
            }
        }
    }
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmW) : "memory");
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&rows_bar[s], CODES ? 1 : m); mbar_init(&empty_bar[s], 1); }
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
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);
    float v[COLS];                                           // the epilogue threads' accumulator rows
    bool ep_ok = true;

    if (warp == 0) {
        // ---- the weights and their scales, and the rows' where they come as codes.  Settled weights fill the ring ahead of the wait
        const uint32_t on = warp_elect(), ring = s_addr(smem);
        const long long g = (long long)e * HALVES + half;
        const uint8_t* sf = sfw + (size_t)(g * ((n + 127) >> 7) + blockIdx.x) * rb_bytes + (size_t)kb0 * MX4_SF_BYTES;
        auto load_w = [&](int s, int i) {
            const uint32_t w_s = ring + s * STAGE_BYTES;
            warp_expect_tx(on, &full_bar[s], TX_BYTES);
            warp_load_2d(on, w_s, &tmW, (kb0 + i) * 128, (int)(g * n) + n0, &full_bar[s]);
            warp_bulk_load(on, w_s + W_BYTES + X_BYTES, sf + (size_t)i * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
        };
        const int head = ahead && !so.offsets ? min(STAGES, my_kb) : 0;
        for (int i = 0; i < head; ++i) load_w(i, i);
        if (!so.offsets) pdl_wait();
        int issued = head, s = 0;
        uint32_t ph = 1;
        for (int i = 0; i < my_kb; ++i) {
            if (i >= head) {
                if (!warp_wait(&empty_bar[s], ph, &abort_flag)) {
                    if (!abort_flag) { atomicExch(err, GR_ERR_EMPTY); abort_flag = 1; }
                    break;
                }
                load_w(s, i);
                issued = i + 1;
            }
            if (CODES) {
                const uint32_t x_s = ring + s * STAGE_BYTES + W_BYTES;
                warp_load_2d(on, x_s, &tmX, (kb0 + i) * 128, r0, &full_bar[s]);
                warp_bulk_load(on, x_s + X_BYTES + MX4_SF_BYTES,
                               reinterpret_cast<const uint8_t*>(X) + (size_t)(r0 >> 7) * rb_bytes + (size_t)(kb0 + i) * MX4_SF_BYTES, MX4_SF_BYTES,
                               &full_bar[s]);
            }
            if (++s == STAGES) { s = 0; ph ^= 1; }
        }
        if (abort_flag) {
            // copies already issued must land before the CTA's shared memory goes away
            volatile int no_abort = 0;
            for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_wait(&full_bar[i % STAGES], (i / STAGES) & 1, &no_abort);
        }
    } else if (warp == 1) {
        // ---- issuer
        const uint32_t on = warp_elect(), ring = s_addr(smem);
        const uint32_t w0 = tile_lo(ring), x0 = tile_lo(ring + W_BYTES), f0 = atom_lo(ring + W_BYTES + X_BYTES);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int i = 0; i < my_kb; ++i) {
            if (!warp_wait(&full_bar[s], ph, &abort_flag) || (!CODES && !warp_wait(&rows_bar[s], ph, &abort_flag))) {
                if (!abort_flag) { atomicExch(err, GR_ERR_FULL); abort_flag = 1; }
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t at = s * (STAGE_BYTES >> 4), f = f0 + at;
            const uint32_t t_w = tmem_base + BN + s * SF_COLS, t_x = t_w + 8;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                tmem_cp_atom<1>(on, t_w + 4 * g, atom_desc(f + g * (MX4_ATOM >> 4)));
                tmem_cp_atom<1>(on, t_x + 4 * g, atom_desc(f + (MX4_SF_BYTES >> 4) + g * (MX4_ATOM >> 4)));
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                umma_mxf4<1>(on, tmem_base, tile_desc(w0 + at + 2 * kk), tile_desc(x0 + at + 2 * kk), idesc_mxf4(128, BN, (kk & 1) * 2),
                             t_w + 4 * (kk >> 1), t_x + 4 * (kk >> 1), (i | kk) != 0);
            umma_done<1>(on, &empty_bar[s]);
            if (++s == STAGES) { s = 0; ph ^= 1; }
        }
        if (ok) umma_done<1>(on, &acc_bar);
    } else if (warp >= 2) {
        // ---- first the rows of X into the stages: warp w takes rows w, w + QW, ... of every stage
        if (!so.offsets) pdl_wait();
        const int first = warp - 2;
        if constexpr (!CODES) if (first < m) {
            RowPart<TX> part[DEPTH][RPW];
            const TX* at[RPW];
#pragma unroll
            for (int j = 0; j < RPW; ++j) {
                const int r = first + QW * j;
                at[j] = X + (r >= m ? 0ll : (so.place ? (long long)s_src[r] : (long long)(r0 + r)) * ldx);
            }
            auto fetch = [&](RowPart<TX> (&p)[RPW], int i) {
                const int col = (kb0 + i) * MX4_CHUNK + lane * 8;
                const bool in = i < my_kb && col < K;
#pragma unroll
                for (int j = 0; j < RPW; ++j) {
                    if (in && first + QW * j < m) p[j].load(at[j] + col);
                    else p[j].zero();
                }
            };
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) fetch(part[d], d);
            bool ok = true;
            for (int ib = 0; ib < my_kb && ok; ib += DEPTH) {
#pragma unroll
                for (int d = 0; d < DEPTH; ++d) {
                    const int i = ib + d, s = i % STAGES;
                    if (i < my_kb && ok) {
                        uint32_t code[RPW], word[RPW];
#pragma unroll
                        for (int j = 0; j < RPW; ++j) {
                            if (j && first + QW * j >= m) break;
                            code[j] = part[d][j].codes(lane, word[j]);
                        }
                        if (!mbar_wait(&empty_bar[s], ((i / STAGES) & 1) ^ 1, &abort_flag)) {
                            if (!abort_flag) { atomicExch(err, GR_ERR_EMPTY); abort_flag = 1; }
                            ok = false;
                        }
                        ok = __all_sync(0xffffffffu, ok);
                        if (ok) {
                            unsigned char* x_s = smem + (size_t)s * STAGE_BYTES + W_BYTES;
                            int mine = 0;
#pragma unroll
                            for (int j = 0; j < RPW; ++j) {
                                const int r = first + QW * j;
                                if (r < m) {
                                    *reinterpret_cast<uint32_t*>(x_s + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2))) = code[j];
                                    if ((lane & 15) == 0)
                                        *reinterpret_cast<uint32_t*>(x_s + X_BYTES + MX4_SF_BYTES + (lane >> 4) * MX4_ATOM +
                                                                     (r & 31) * 16 + (r >> 5) * 4) = word[j];
                                    ++mine;
                                }
                            }
                            fence_async_smem();
                            __syncwarp();
                            if (lane < mine) mbar_arrive(&rows_bar[s]);        // one arrival for every row
                        }
                    }
                    fetch(part[d], i + DEPTH);
                }
            }
        }
        // ---- then the accumulator (thread = weight row, registers = rows of X: all of them, or with eight warps half)
        const int q = warp & 3, row = q * 32 + lane, b_first = ((warp - 2) >> 2) * COLS;
        ep_ok = mbar_wait(&acc_bar, 0, &abort_flag);
        if (!ep_ok && !abort_flag) { atomicExch(err, GR_ERR_ACC); abort_flag = 1; }
        ep_ok = __all_sync(0xffffffffu, ep_ok);
        pdl_launch_dependents();
        if (ep_ok) {
            tc_fence_after();
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + b_first;
#pragma unroll
            for (int c0 = 0; c0 < COLS; c0 += 16) tmem_ld16(taddr + c0, v + c0);
            tmem_ld_wait();
        } else {
#pragma unroll
            for (int b = 0; b < COLS; ++b) v[b] = 0.f;
        }
        if (ranks > 1) {
#pragma unroll
            for (int b = 0; b < COLS; ++b)
                if (b_first + b < m) red[(b_first + b) * 128 + row] = v[b];
        }
    }
    __syncwarp();          // the lanes that had no role meet the elected one: the barriers below want whole warps
    tc_fence_before();
    __syncthreads();
    // NB rows of X at a column of C, from b0 in steps of `step`
    constexpr int NB = 8;
    const Mx4Glu unit(glu);
    auto write = [&](int b0, int step, int col, const float (&sum)[HALVES][NB]) {
        if (col >= n || !ep_ok) return;
        TC* dst = C + (size_t)(r0 + b0) * ldc + col;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const float o = !GATED ? sum[0][i] : unit.gelu ? unit.template at<true>(sum[0][i], sum[HALVES - 1][i]) : unit.template at<false>(sum[0][i], sum[HALVES - 1][i]);
            if (b0 + i * step < m) {
                if constexpr (EPI == GR_EPI_ACCUM) add_to(dst + (size_t)(i * step) * ldc, o);
                else dst[(size_t)(i * step) * ldc] = from_f<TC>(o);
            }
        }
    };
    if (ranks > 1) {
        // every thread of every CTA of the cluster comes here, whatever happened before.  #1: all sums are parked
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (warp >= 2) {
            // this CTA's 128 / ranks weight rows; the groups of as many threads take the rows of X in turn
            const int t = tid - 64, share = 128 / ranks, groups = QW / 4 * ranks, row = (int)blockIdx.y * share + (t & (share - 1));
            for (int b0 = t / share; b0 < m; b0 += NB * groups) {
                float sum[HALVES][NB];
                for (int z = 0; z < n_splits; ++z) {             // in rank order: ascending k
                    float f[HALVES][NB];
#pragma unroll
                    for (int w = 0; w < HALVES; ++w) {
                        uint32_t remote;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(s_addr(red + row)), "r"(w * n_splits + z));
#pragma unroll
                        for (int i = 0; i < NB; ++i) {
                            const int b = b0 + i * groups;
                            f[w][i] = 0.f;
                            if (b < m) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[w][i]) : "r"(remote + (uint32_t)b * 512u) : "memory");
                        }
                    }
#pragma unroll
                    for (int w = 0; w < HALVES; ++w)
#pragma unroll
                        for (int i = 0; i < NB; ++i) sum[w][i] = z ? sum[w][i] + f[w][i] : f[w][i];
                }
                write(b0, groups, n0 + row, sum);
            }
        }
        __syncwarp();      // the lanes' rows of X may have ended at different turns
        // #2: nobody reads another CTA's shared memory any more
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else if (warp >= 2) {
        const int row = (warp & 3) * 32 + lane, b_first = ((warp - 2) >> 2) * COLS;
#pragma unroll
        for (int b0 = 0; b0 < COLS; b0 += NB) {
            float sum[HALVES][NB];
#pragma unroll
            for (int i = 0; i < NB; ++i) sum[0][i] = sum[HALVES - 1][i] = v[b0 + i];
            if (b_first + b0 < m) write(b_first + b0, 1, n0 + row, sum);
        }
    }
    if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

// ---------------------------------------------------------------- host side
template <int BN, int STAGES, int QW, int CTAS, int EPI, typename TC, typename TX>
static int gr_launch(const CUtensorMap& tw, const CUtensorMap& tx, const void* sfw, const void* X, long long ldx, void* C, long long ldc, int m, int n, int K,
                     int ahead, const GluForm glu, const GrSorted& so, int splits, int* err, cudaStream_t stream) {
    constexpr int STAGE_BYTES = 128 * 128 + BN * 128 + 2 * MX4_SF_BYTES, smem = STAGES * STAGE_BYTES + 1024;
    static_assert(BN * 128 * 4 <= STAGES * STAGE_BYTES, "parked sums fit the stages");
    auto kern = gemm_mx4_rows_kernel<BN, STAGES, QW, CTAS, EPI, TC, TX>;
    const int st = mx4_allow_smem(kern, smem);
    if (st) return st;
    // chunks of rows: with experts at most one begun chunk for each expert that can have rows beside the full ones
    const long long chunks = so.offsets ? (long long)m / BN + (m < so.E ? m : so.E) : ((long long)m + BN - 1) / BN;
    const int ranks = splits * (EPI == GR_EPI_GATED ? 2 : 1);
    if (chunks > 65535) return (int)cudaErrorInvalidValue;
    return rllm_launch_cluster(kern, dim3((n + 127) / 128, ranks, (unsigned)chunks), dim3(64 + 32 * QW), smem, stream, ranks, tw, tx,
                               (const uint8_t*)sfw, (const TX*)X, ldx, (TC*)C, ldc, m, n, K, ahead, glu, so, err);
}

// mx4.cu
RLLM_API int rllm_mx4_quantize(const void* x, void* codes, void* scales, const int* offsets, const int* place, long long ld, int dt,
                               int rows, int k, int pad, int E, int top_k, cudaStream_t stream);

// X: rows of K entries, ldx apart, float32 or bfloat16; C [m, n].  W: codes [n, K / 2] and scales, gated: gate and up matrix of n rows each,
// experts: E times that.  bn: rows of X to a CTA.  16: they are quantised by the product itself (16-byte aligned rows); 32, 64 (all rows in
// one chunk) and 128 (not gated): by a launch ahead of it, into `work` (codes, and from the next multiple of 1,024 bytes the scales).  splits: 1, 2, 4
// or 8 CTAs (gated: pairs, up to 4) share a tile's K.  offsets, place, top_k: see the top (bn 16; place: X holds m / top_k rows).  ahead: W is
// settled and may be read before the kernels before have ended.  epilogue 0 store, 1 add into a float32 C, 2 gated (GluForm).  Returns 0, a
// cudaError_t or 30000 + CUresult.
RLLM_API int rllm_mx4_rows_product(const void* X, const int* offsets, const int* place, const void* w_codes, const void* w_scales, void* C,
                                   void* work, int* err, long long ldx, long long ldc, int x_dtype, int c_dtype, int m, int n, int K, int E,
                                   int top_k, int epilogue, int bn, int splits, int ahead, float glu_limit, float glu_alpha, float glu_shift,
                                   cudaStream_t stream) {
    if (m <= 0 || n <= 0) return 0;
    const bool gated = epilogue == GR_EPI_GATED;
    const long long matrices = (long long)(offsets ? E : 1) * (gated ? 2 : 1);
    if (K <= 0 || (K % MX4_BLOCK) || !err || ldc < n || matrices * n > 0x7fffff00LL || m > 0x7fffff00 || ((uintptr_t)w_codes & 15) ||
        ((uintptr_t)w_scales & 15) || (bn == 16 && (((uintptr_t)X & 15) || ((ldx * (x_dtype == RLLM_F32 ? 4 : 2)) & 15))) ||
        (splits != 1 && splits != 2 && splits != 4 && (splits != 8 || gated)) || splits > (K + MX4_CHUNK - 1) / MX4_CHUNK ||
        (epilogue == GR_EPI_ACCUM && (c_dtype != RLLM_F32 || offsets)) || (offsets && (E <= 0 || bn != 16)) ||
        (place && (!offsets || top_k <= 0)) || (bn != 16 && (!work || ((uintptr_t)work & 15))) || (bn < 128 && bn != 16 && m > bn))
        return (int)cudaErrorInvalidValue;
    CUtensorMap tw, tx = {};
    int st = mx4_tmap(&tw, w_codes, matrices * n, K, 128);
    if (st) return st;
    const void* rows = X;
    if (bn != 16) {
        unsigned char* scales = (unsigned char*)work + (((size_t)m * (size_t)(K / 2) + 1023) & ~(size_t)1023);
        st = rllm_mx4_quantize(X, work, scales, nullptr, nullptr, ldx, x_dtype, m, K, 0, 0, 0, stream);
        if (st) return st;
        st = mx4_tmap(&tx, work, m, K, bn);
        if (st) return st;
        rows = scales;
    }
    const GluForm glu = GluForm{glu_limit, glu_alpha, glu_shift};
    const GrSorted so = {offsets, place, E, top_k, m};
#define GR_GO(BN, ST, QW, CT, EPI, TC, TX) \
    return gr_launch<BN, ST, QW, CT, EPI, TC, TX>(tw, tx, w_scales, rows, ldx, C, ldc, m, n, K, ahead, glu, so, splits, err, stream)
#define GR_BN(EPI, TC)                                                                                          \
    {                                                                                                           \
        if (bn == 16 && x_dtype == RLLM_F32) { GR_GO(16, 3, 4, 3, EPI, TC, float); }                            \
        if (bn == 16) { GR_GO(16, 3, 4, 3, EPI, TC, bf16); }                                                    \
        if (bn == 32) { GR_GO(32, 3, 4, 3, EPI, TC, uint8_t); }                                                 \
        if (bn == 64) { GR_GO(64, 4, 8, 2, EPI, TC, uint8_t); }                                                 \
    }
#define GR_128(EPI, TC) if (bn == 128) { GR_GO(128, 3, 8, 2, EPI, TC, uint8_t); }
    if (epilogue == GR_EPI_STORE && c_dtype == RLLM_F32) { GR_BN(GR_EPI_STORE, float) GR_128(GR_EPI_STORE, float) }
    if (epilogue == GR_EPI_STORE && c_dtype != RLLM_F32) { GR_BN(GR_EPI_STORE, bf16) GR_128(GR_EPI_STORE, bf16) }
    if (epilogue == GR_EPI_ACCUM) { GR_BN(GR_EPI_ACCUM, float) GR_128(GR_EPI_ACCUM, float) }
    if (gated) { if (c_dtype == RLLM_F32) GR_BN(GR_EPI_GATED, float) else GR_BN(GR_EPI_GATED, bf16) }
#undef GR_128
#undef GR_BN
#undef GR_GO
    return (int)cudaErrorInvalidValue;
}

TC_DEFINE_WAIT_CONTROLS(rllm_gemm_mx4_rows)

RLLM_PACKED(rllm_mx4_rows_product)
