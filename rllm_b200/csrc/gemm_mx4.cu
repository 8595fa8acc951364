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
//     back before they convert and store (handed back before it was read, a launch took as long: the stores cost, not the hand-over).
// A stage's four products need 512 cycles: 0.27 us at 1.9 GHz, 0.31 at the 1.68 GHz that long launches run at under the power cap; a stage takes 0.41 us
// (in pairs, below, 0.31 to 0.38).  The copies of the scales are not what is missing: with half of them left out it took as long.  Gated 256 x 1,536 x 2,048: 8.8 us with the quantisation of the rows ahead of it; 4,000 rows of 16 experts, 2 x 768 x
// 2,048: 15.5 us of 19.9.  Where K is short the tile's end decides: its rows leave as whole lines (gm_give).
// The rows of A may be sorted by expert (offsets int32 [E + 1] on the device): expert e's rows form row tiles of their own, counted by
// every CTA itself, whose scales lie in the same order (rllm_mx4_quantize); its matrix is number e of the stack B.
// The gated product: B is a stack of gate and up matrices in turn; a tile holds 128 gate rows and the 128 up rows of the same index.
#include "mx4_tc.cuh"

// mx4.cu
RLLM_API int rllm_mx4_quantize(const void* x, void* codes, void* scales, const int* offsets, const int* place, long long ld, int dt,
                               int rows, int k, int pad, int E, int top_k, cudaStream_t stream);

#define GM_BM 128
#define GM_BN 256
#define GM_STAGES 3
#define GM_THREADS 320
#define GM_MAX_E 1024
#define GM_A_BYTES (GM_BM * 128)
#define GM_B_BYTES (GM_BN * 128)
#define GM_STAGE_BYTES (GM_A_BYTES + GM_B_BYTES + 3 * MX4_SF_BYTES)
#define GM_SF_COLS 32                                      // tensor-memory columns of a stage's scales: 8 of A, 16 of B

enum { GM_EPI_STORE = 0, GM_EPI_ACCUM = 1, GM_EPI_GATED = 2 };
enum { GM_ERR_FULL = 31, GM_ERR_EMPTY = 32, GM_ERR_ACC = 33 };

// A thread's half of an accumulator row into registers: 128 columns, gated 64 gate columns and the 64 up columns of the same index.
template <bool GATED> __device__ __forceinline__ void gm_take(uint32_t taddr, int half, uint32_t (&r)[4][32]) {
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
}
// ... and from there to C.  A thread holds columns of one row; written as they are, 16 bytes a thread, a store would touch 32 lines, and the
// stores of a tile of 128 x 256 float32 would take longer than its products at K 2,000.  So the warp's 32 rows pass through 4 KB of shared
// memory, 128 bytes of each at a time (pieces of 16 bytes swizzled by the row), and leave as whole lines, eight lanes to a row.
//   row0: the warp's first row, n0: the first column of what its threads hold, `vec`: rows of C begin at multiples of 16 bytes
template <typename TC, int EPI> __device__ __forceinline__ void gm_give(const uint32_t (&r)[4][32], unsigned char* stage, int lane, TC* C, long long ldc,
                                                                        int row0, int m_end, int n0, int N, bool vec, const Mx4Glu& glu) {
    constexpr bool GATED = EPI == GM_EPI_GATED;
    constexpr int PER = 128 / (int)sizeof(TC), PIECE = 16 / (int)sizeof(TC), OUT = GATED ? 64 : 128;
#pragma unroll
    for (int c = 0; c < OUT / PER; ++c) {
        if (n0 + c * PER >= N) break;
        auto pieces = [&](auto value) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float v[PIECE];
#pragma unroll
                for (int i = 0; i < PIECE; ++i) v[i] = value(c * PER + j * PIECE + i);
                uint4 u;
                if constexpr (sizeof(TC) == 4) u = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                else {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                        w[i] = *reinterpret_cast<const uint32_t*>(&b);
                    }
                    u = make_uint4(w[0], w[1], w[2], w[3]);
                }
                *reinterpret_cast<uint4*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = u;
            }
        };
        if constexpr (GATED) {
            auto gate = [&](int col) { return __uint_as_float(r[col >> 5][col & 31]); };
            auto up = [&](int col) { return __uint_as_float(r[(col >> 5) + 2][col & 31]); };
            if (glu.gelu) pieces([&](int col) { return glu.template at<true>(gate(col), up(col)); });
            else pieces([&](int col) { return glu.template at<false>(gate(col), up(col)); });
        } else {
            pieces([&](int col) { return __uint_as_float(r[col >> 5][col & 31]); });
        }
        __syncwarp();
        if (vec && n0 + (c + 1) * PER <= N) {
            const int col = n0 + c * PER + (lane & 7) * PIECE;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = i * 4 + (lane >> 3), gm = row0 + row;
                const uint4 u = *reinterpret_cast<const uint4*>(stage + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
                if (gm < m_end) {
                    TC* dst = C + (size_t)gm * ldc + col;
                    if constexpr (EPI == GM_EPI_ACCUM) add_to4(dst, u);
                    else *reinterpret_cast<uint4*>(dst) = u;
                }
            }
        } else {                                     // rows at any address, columns that end inside: a row at a time, neighbouring lanes side by side
            for (int row = 0; row < 32 && row0 + row < m_end; ++row) {
                TC* dst = C + (size_t)(row0 + row) * ldc + n0 + c * PER;
#pragma unroll
                for (int h = 0; h < PER / 32; ++h) {
                    const int at = h * 32 + lane, piece = at / PIECE;
                    const TC v = *reinterpret_cast<const TC*>(stage + row * 128 + ((piece ^ (row & 7)) << 4) + (at & (PIECE - 1)) * (int)sizeof(TC));
                    if (n0 + c * PER + at < N) {
                        if constexpr (EPI == GM_EPI_ACCUM) add_to(dst + at, v);
                        else dst[at] = v;
                    }
                }
            }
        }
        __syncwarp();
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

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
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
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);
    const int m_tiles = __shfl_sync(0xffffffffu, s_tile[E], 0), total_tiles = m_tiles * n_tiles;
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

    if (warp == 0) {
        // ---- producer: one continuous ring over all of this CTA's tiles
        const uint32_t on = warp_elect(), ring = s_addr(smem);
        int s = 0, issued = 0;
        uint32_t ph = 1;
        bool ok = true;
        auto load_b = [&](int s, int kb, int e, int n0) {
            const uint32_t b_s = ring + s * GM_STAGE_BYTES + GM_A_BYTES, f_s = b_s + GM_B_BYTES + MX4_SF_BYTES;
            const int rb = n0 >> 7;
            if (GATED) {
                const long long g = 2ll * e;
                warp_load_2d(on, b_s, &tmB, kb * 128, (int)(g * N) + n0, &full_bar[s]);
                warp_load_2d(on, b_s + GM_B_BYTES / 2, &tmB, kb * 128, (int)((g + 1) * N) + n0, &full_bar[s]);
                warp_bulk_load(on, f_s, sfb + (g * rb_n + rb) * rb_bytes + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
                warp_bulk_load(on, f_s + MX4_SF_BYTES, sfb + ((g + 1) * rb_n + rb) * rb_bytes + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES,
                               &full_bar[s]);
            } else {
                // (the second 128 rows of a matrix's last tile may not exist: whatever comes in belongs to columns that are dropped)
                const long long r0 = (long long)e * rb_n;
                warp_load_2d(on, b_s, &tmB, kb * 128, e * N + n0, &full_bar[s]);
                warp_load_2d(on, b_s + GM_B_BYTES / 2, &tmB, kb * 128, e * N + n0 + 128, &full_bar[s]);
                warp_bulk_load(on, f_s, sfb + (r0 + rb) * rb_bytes + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
                warp_bulk_load(on, f_s + MX4_SF_BYTES, sfb + (r0 + min(rb + 1, rb_n - 1)) * rb_bytes + (size_t)kb * MX4_SF_BYTES,
                               MX4_SF_BYTES, &full_bar[s]);
            }
        };
        // weights that are settled do not depend on the kernel before: the first stages' start ahead of the wait
        int head = ahead && !offsets && (int)blockIdx.x < total_tiles ? min(GM_STAGES, nkb) : 0;
        if (head) {
            int e, mt, m0, m_end, n0;
            place(blockIdx.x, e, mt, m0, m_end, n0);
            for (int i = 0; i < head; ++i) {
                warp_expect_tx(on, &full_bar[i], GM_STAGE_BYTES);
                load_b(i, i, e, n0);
            }
        }
        if (!offsets) pdl_wait();
        for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x) {
            int e, mt, m0, m_end, n0;
            place(tile, e, mt, m0, m_end, n0);
            const uint8_t* sf_rows = sfa + (size_t)min(mt, rb_most - 1) * rb_bytes;
            for (int kb = 0; kb < nkb; ++kb) {
                if (!warp_wait(&empty_bar[s], ph, &abort_flag)) {
                    if (!abort_flag) { atomicExch(err, GM_ERR_EMPTY); abort_flag = 1; }
                    ok = false;
                    break;
                }
                const uint32_t a_s = ring + s * GM_STAGE_BYTES;
                if (head == 0) warp_expect_tx(on, &full_bar[s], GM_STAGE_BYTES);
                warp_load_2d(on, a_s, &tmA, kb * 128, m0, &full_bar[s]);
                warp_bulk_load(on, a_s + GM_A_BYTES + GM_B_BYTES, sf_rows + (size_t)kb * MX4_SF_BYTES, MX4_SF_BYTES, &full_bar[s]);
                if (head == 0) load_b(s, kb, e, n0);
                else --head;
                ++issued;
                if (++s == GM_STAGES) { s = 0; ph ^= 1; }
            }
        }
        if (abort_flag) {
            // copies already issued must land before the CTA's shared memory goes away
            volatile int no_abort = 0;
            for (int i = max(0, issued - GM_STAGES); i < issued; ++i)
                mbar_wait(&full_bar[i % GM_STAGES], (i / GM_STAGES) & 1, &no_abort);
        }
    } else if (warp == 1) {
        // ---- issuer: the stage's scales to tensor memory, then four products of 64 entries along K
        const uint32_t on = warp_elect(), ring = s_addr(smem);
        const uint32_t a0 = tile_lo(ring), b0 = tile_lo(ring + GM_A_BYTES), f0 = atom_lo(ring + GM_A_BYTES + GM_B_BYTES);
        int s = 0, local = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x, ++local) {
            if (!warp_wait(&acc_empty, (local & 1) ^ 1, &abort_flag)) {
                if (!abort_flag) { atomicExch(err, GM_ERR_ACC); abort_flag = 1; }
                break;
            }
            tc_fence_after();
            for (int kb = 0; kb < nkb; ++kb) {
                if (!warp_wait(&full_bar[s], ph, &abort_flag)) {
                    if (!abort_flag) { atomicExch(err, GM_ERR_FULL); abort_flag = 1; }
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t at = s * (GM_STAGE_BYTES >> 4), f = f0 + at;
                const uint32_t t_a = tmem_base + GM_BN + s * GM_SF_COLS, t_b = t_a + 8;
#pragma unroll
                for (int g = 0; g < 2; ++g) {                // 128 entries along K each
                    tmem_cp_atom<1>(on, t_a + 4 * g, atom_desc(f + g * (MX4_ATOM >> 4)));
                    tmem_cp_atom<1>(on, t_b + 8 * g, atom_desc(f + (MX4_SF_BYTES >> 4) + g * (MX4_ATOM >> 4)));
                    tmem_cp_atom<1>(on, t_b + 8 * g + 4, atom_desc(f + 2 * (MX4_SF_BYTES >> 4) + g * (MX4_ATOM >> 4)));
                }
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)               // 64 entries = 32 bytes along K: +2 in 16-byte units
                    umma_mxf4<1>(on, tmem_base, tile_desc(a0 + at + 2 * kk), tile_desc(b0 + at + 2 * kk), idesc_mxf4(GM_BM, GM_BN, (kk & 1) * 2),
                                 t_a + 4 * (kk >> 1), t_b + 8 * (kk >> 1), (kb | kk) != 0);
                umma_done<1>(on, &empty_bar[s]);
                if (++s == GM_STAGES) { s = 0; ph ^= 1; }
            }
            if (ok) umma_done<1>(on, &acc_full);
        }
    } else if (warp >= 2) {
        // ---- epilogue: warp w may touch the lanes 32 * (w % 4) .. + 31; the first four take the first half of the columns
        if (!offsets) pdl_wait();
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        unsigned char* stage = smem + GM_STAGES * GM_STAGE_BYTES + (warp - 2) * 4096;
        const bool vec = ((uintptr_t)C & 15) == 0 && ((ldc * (long long)sizeof(TC)) & 15) == 0;
        const Mx4Glu unit(glu);
        int local = 0;
        for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++local) {
            int e, mt, m0, m_end, n0;
            place(tile, e, mt, m0, m_end, n0);
            bool ok = mbar_wait(&acc_full, local & 1, &abort_flag);
            if (!ok && !abort_flag) { atomicExch(err, GM_ERR_ACC); abort_flag = 1; }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            if (tile + (int)gridDim.x >= total_tiles) pdl_launch_dependents();
            uint32_t r[4][32];
            gm_take<GATED>(tmem_base + ((uint32_t)(quarter * 32) << 16), half, r);
            tc_fence_before();
            mbar_arrive(&acc_empty);
            if (m0 + quarter * 32 < m_end)
                gm_give<TC, EPI>(r, stage, lane, C, ldc, m0 + quarter * 32, m_end, n0 + (GATED ? 64 : 128) * half, N, vec, unit);
        }
    }
    __syncwarp();          // the lanes that had no role meet the elected one: the barrier below wants whole warps
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// ---------------------------------------------------------------- two SMs to a tile
// The same product by pairs of CTAs (tcgen05.mma.cta_group::2, a cluster of two along x): a pair computes 256 x 256, each CTA stages its own
// 128 rows of A and its half of the tile of B, and holds the accumulator of its rows.  A stage of 256 entries along K is then 35 KB a CTA where the
// kernel above fills 51, and five stages fit.  2,048 x 4,096 x 12,288: 40 us behind 12 of quantisation, 5.2 PFLOP/s (61 us together with one SM a tile, 52
// with two); gated 2,048 x 2 x 12,288 x 4,096: 80 us, 5.2 PFLOP/s.
//   * the scales of A belong to each CTA's own rows; those of B are needed whole by both, so each loads both blocks;
//   * the loads of both CTAs complete on the leader's barrier; a plain bulk copy cannot signal the peer's barrier, so the scales, too, come by
//     tensor loads, from a map of lines of 1,024 bytes;
//   * tcgen05.cp.cta_group::2 spreads the scales of each CTA's shared memory over its own tensor memory.
#define GP_STAGES 5
#define GP_STAGE_BYTES (2 * GM_A_BYTES + 3 * MX4_SF_BYTES)          // A, half of B, scales of A, scales of B

__device__ __forceinline__ uint32_t gp_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t gp_leader(const void* p) {      // the leader's copy of `p` in the cluster's shared window
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(s_addr(p)));
    return a;
}
__device__ __forceinline__ void gp_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
struct GpMaps { CUtensorMap a, b, sfa, sfb; };

template <typename TC, int EPI>
__global__ void __launch_bounds__(GM_THREADS, 1)
gemm_mx4_pair_kernel(const __grid_constant__ GpMaps maps, TC* C, long long ldc, const int* offsets, int E, int rows, int N, int K,
                     const GluForm glu, int* err) {
    constexpr bool GATED = EPI == GM_EPI_GATED;
    constexpr int BN_OUT = GATED ? GM_BN / 2 : GM_BN;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t full_bar[GP_STAGES];      // used in the leader: bytes of both CTAs
    __shared__ __align__(8) uint64_t empty_bar[GP_STAGES];     // in each CTA: the products have read the stage
    __shared__ __align__(8) uint64_t acc_full;                 // in each CTA
    __shared__ __align__(8) uint64_t acc_empty;                // used in the leader: the eight epilogue warps of both CTAs
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    __shared__ int s_row[GM_MAX_E + 1];              // an expert's first row,
    __shared__ int s_tile[GM_MAX_E + 1];             // its first row tile (of 256)
    __shared__ int s_block[GM_MAX_E + 1];            // and its first block of 128 scale rows

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int rank = (int)gp_rank(), pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const int nkb = (K + MX4_CHUNK - 1) / MX4_CHUNK, n_tiles = (N + BN_OUT - 1) / BN_OUT, rb_n = (N + 127) >> 7;
    const int rb_most = (rows + GM_BM - 1) / GM_BM + (offsets ? E : 0);
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.b) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.sfa) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.sfb) : "memory");
        for (int s = 0; s < GP_STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        mbar_init(&acc_full, 1);
        mbar_init(&acc_empty, 16);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s_addr(&tmem_base_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pdl_wait();                                      // rows and offsets are written by the kernels before
    if (warp == 2) {                                 // the experts' first rows, tiles and scale blocks, 32 at a time
        int tiles = 0, blocks = 0;
        for (int e0 = 0; e0 <= E; e0 += 32) {
            const int e = e0 + lane;
            const int first = e > E ? 0 : offsets ? min(max(offsets[e], 0), rows) : (e == 0 ? 0 : rows);
            const int next = e >= E ? first : offsets ? min(max(offsets[e + 1], 0), rows) : rows;
            const int count = e < E ? max(next - first, 0) : 0, t = (count + 2 * GM_BM - 1) / (2 * GM_BM), b = (count + GM_BM - 1) / GM_BM;
            int it = t, ib = b;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const int ut = __shfl_up_sync(0xffffffffu, it, m), ub = __shfl_up_sync(0xffffffffu, ib, m);
                if (lane >= m) { it += ut; ib += ub; }
            }
            if (e <= E) {
                s_row[e] = first;
                s_tile[e] = min(tiles + it - t, rb_most);
                s_block[e] = blocks + ib - b;
            }
            tiles += __shfl_sync(0xffffffffu, it, 31);
            blocks += __shfl_sync(0xffffffffu, ib, 31);
        }
    }
    tc_fence_before();
    __syncthreads();
    gp_sync();                                       // the peer's barriers exist before anything arrives at them
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);
    const int m_tiles = __shfl_sync(0xffffffffu, s_tile[E], 0), total_tiles = m_tiles * n_tiles;
    // tile -> its expert, this CTA's first row and block of scale rows, rows of the expert from there on, first column
    auto place = [&](int tile, int& e, int& block, int& m0, int& m_end, int& n0) {
        const int mt = tile % m_tiles;
        int lo = 0, hi = E;                          // the last expert whose first tile is <= mt (and that has tiles)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_tile[mid] <= mt) lo = mid; else hi = mid;
        }
        e = lo;
        const int sub = 2 * (mt - s_tile[lo]) + rank;
        block = s_block[lo] + sub;
        m0 = s_row[lo] + sub * GM_BM;
        m_end = s_row[lo + 1];
        n0 = tile / m_tiles * BN_OUT;
    };

    if (warp == 0) {
        // ---- producer of this CTA: its rows of A, its half of B, and the scales
        const uint32_t on = warp_elect(), ring = s_addr(smem), full0 = gp_leader(full_bar);
        int s = 0, issued = 0;
        uint32_t ph = 1;
        bool ok = true;
        for (int tile = pair; tile < total_tiles && ok; tile += n_pairs) {
            int e, block, m0, m_end, n0;
            place(tile, e, block, m0, m_end, n0);
            const int b_row = GATED ? (2 * e + rank) * N + n0 : e * N + n0 + rank * 128;
            const int sa = min(block, rb_most - 1) * nkb, rb = n0 >> 7;
            const int sb0 = (GATED ? 2 * e * rb_n + rb : e * rb_n + rb) * nkb;
            const int sb1 = (GATED ? (2 * e + 1) * rb_n + rb : e * rb_n + min(rb + 1, rb_n - 1)) * nkb;
            for (int kb = 0; kb < nkb; ++kb) {
                if (!warp_wait(&empty_bar[s], ph, &abort_flag)) {
                    if (!abort_flag) { atomicExch(err, GM_ERR_EMPTY); abort_flag = 1; }
                    ok = false;
                    break;
                }
                const uint32_t a_s = ring + s * GP_STAGE_BYTES, f_s = a_s + 2 * GM_A_BYTES, full = full0 + 8 * s;
                if (rank == 0) warp_expect_tx(on, &full_bar[s], 2 * GP_STAGE_BYTES);
                warp_load_2d_pair(on, a_s, &maps.a, kb * 128, m0, full);
                warp_load_2d_pair(on, a_s + GM_A_BYTES, &maps.b, kb * 128, b_row, full);
                warp_load_2d_pair(on, f_s, &maps.sfa, 0, sa + kb, full);
                warp_load_2d_pair(on, f_s + MX4_SF_BYTES, &maps.sfb, 0, sb0 + kb, full);
                warp_load_2d_pair(on, f_s + 2 * MX4_SF_BYTES, &maps.sfb, 0, sb1 + kb, full);
                ++issued;
                if (++s == GP_STAGES) { s = 0; ph ^= 1; }
            }
        }
        if (abort_flag && rank == 0) {
            // copies already issued must land before the shared memory goes away (the peer's land in its own; both CTAs stay until the
            // cluster barrier at the end)
            volatile int no_abort = 0;
            for (int i = max(0, issued - GP_STAGES); i < issued; ++i)
                mbar_wait(&full_bar[i % GP_STAGES], (i / GP_STAGES) & 1, &no_abort);
        }
    } else if (warp == 1) {
        // ---- issuer of the pair, in the leader
        const uint32_t on = warp_elect(), ring = s_addr(smem);
        const uint32_t a0 = tile_lo(ring), b0 = tile_lo(ring + GM_A_BYTES), f0 = atom_lo(ring + 2 * GM_A_BYTES);
        int s = 0, local = 0;
        uint32_t ph = 0;
        bool ok = rank == 0;
        for (int tile = pair; tile < total_tiles && ok; tile += n_pairs, ++local) {
            if (!warp_wait(&acc_empty, (local & 1) ^ 1, &abort_flag)) {
                if (!abort_flag) { atomicExch(err, GM_ERR_ACC); abort_flag = 1; }
                break;
            }
            tc_fence_after();
            for (int kb = 0; kb < nkb; ++kb) {
                if (!warp_wait(&full_bar[s], ph, &abort_flag)) {
                    if (!abort_flag) { atomicExch(err, GM_ERR_FULL); abort_flag = 1; }
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t at = s * (GP_STAGE_BYTES >> 4), f = f0 + at;
                const uint32_t t_a = tmem_base + GM_BN + s * GM_SF_COLS, t_b = t_a + 8;
#pragma unroll
                for (int g = 0; g < 2; ++g) {                // 128 entries along K each
                    tmem_cp_atom<2>(on, t_a + 4 * g, atom_desc(f + g * (MX4_ATOM >> 4)));
                    tmem_cp_atom<2>(on, t_b + 8 * g, atom_desc(f + (MX4_SF_BYTES >> 4) + g * (MX4_ATOM >> 4)));
                    tmem_cp_atom<2>(on, t_b + 8 * g + 4, atom_desc(f + 2 * (MX4_SF_BYTES >> 4) + g * (MX4_ATOM >> 4)));
                }
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    umma_mxf4<2>(on, tmem_base, tile_desc(a0 + at + 2 * kk), tile_desc(b0 + at + 2 * kk), idesc_mxf4(2 * GM_BM, GM_BN, (kk & 1) * 2),
                                 t_a + 4 * (kk >> 1), t_b + 8 * (kk >> 1), (kb | kk) != 0);
                umma_done<2>(on, &empty_bar[s]);
                if (++s == GP_STAGES) { s = 0; ph ^= 1; }
            }
            if (ok) umma_done<2>(on, &acc_full);
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        unsigned char* stage = smem + GP_STAGES * GP_STAGE_BYTES + (warp - 2) * 4096;
        const bool vec = ((uintptr_t)C & 15) == 0 && ((ldc * (long long)sizeof(TC)) & 15) == 0;
        const Mx4Glu unit(glu);
        int local = 0;
        for (int tile = pair; tile < total_tiles; tile += n_pairs, ++local) {
            int e, block, m0, m_end, n0;
            place(tile, e, block, m0, m_end, n0);
            bool ok = mbar_wait(&acc_full, local & 1, &abort_flag);
            if (!ok && !abort_flag) { atomicExch(err, GM_ERR_ACC); abort_flag = 1; }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            if (tile + n_pairs >= total_tiles) pdl_launch_dependents();
            uint32_t r[4][32];
            gm_take<GATED>(tmem_base + ((uint32_t)(quarter * 32) << 16), half, r);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(gp_leader(&acc_empty)) : "memory");
            if (m0 + quarter * 32 < m_end)
                gm_give<TC, EPI>(r, stage, lane, C, ldc, m0 + quarter * 32, m_end, n0 + (GATED ? 64 : 128) * half, N, vec, unit);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    gp_sync();             // the leader's products read the peer's shared memory and arrive at its barriers: leave together
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
}

// ---------------------------------------------------------------- host side
// A: codes [rows, K / 2] and scales; B: codes [matrices * N, K / 2] and the matrices' scales one after another (matrices: E, gated
// 2 E, gate and up in turn).  K a multiple of 32, all bases 16-byte aligned.  offsets int32 [E + 1] on the device (null: E is 1, all
// rows are its).  epilogue 0 store, 1 add into a float32 C, 2 gated (GluForm).  pairs: two SMs to a tile.  ahead: B is settled and may be read before the
// kernels before have ended.  Returns 0, a cudaError_t or 30000 + CUresult of the tensor-map encoder.
static int rllm_gemm_mx4(const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales, void* C, int c_dtype,
                           long long ldc, const int* offsets, int E, int rows, int N, int K, int epilogue, int pairs, int ahead,
                           float glu_limit, float glu_alpha, float glu_shift, int* err, cudaStream_t stream) {
    if (rows <= 0 || N <= 0) return 0;
    const long long matrices = (long long)E * (epilogue == GM_EPI_GATED ? 2 : 1);
    if (E <= 0 || E > GM_MAX_E || (!offsets && E != 1) || K <= 0 || (K % MX4_BLOCK) || !err || ldc < N || matrices * N > 0x7fffff00LL ||
        rows > 0x7fffff00 || ((uintptr_t)a_codes & 15) || ((uintptr_t)a_scales & 15) || ((uintptr_t)b_codes & 15) ||
        ((uintptr_t)b_scales & 15) || (epilogue == GM_EPI_ACCUM && c_dtype != RLLM_F32))
        return (int)cudaErrorInvalidValue;
    const GluForm glu = GluForm{glu_limit, glu_alpha, glu_shift};
    const int bn_out = epilogue == GM_EPI_GATED ? GM_BN / 2 : GM_BN, n_sm = rllm_sm_count();
    const int tile_rows = pairs ? 2 * GM_BM : GM_BM;
    const long long most = ((long long)(rows + tile_rows - 1) / tile_rows + (offsets ? E : 0)) * ((N + bn_out - 1) / bn_out);
    const long long blocks_a = (rows + 127) / 128 + (offsets ? E : 0), blocks_b = matrices * ((N + 127) / 128), nkb = (K + MX4_CHUNK - 1) / MX4_CHUNK;
    if (most > 0x7fffffffLL || blocks_a * nkb > 0x7fffffffLL || blocks_b * nkb > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    GpMaps maps;
    int st = mx4_tmap(&maps.a, a_codes, rows, K, GM_BM);
    if (!st) st = mx4_tmap(&maps.b, b_codes, matrices * N, K, 128);
    if (!st && pairs) st = mx4_scale_tmap(&maps.sfa, a_scales, blocks_a * nkb);
    if (!st && pairs) st = mx4_scale_tmap(&maps.sfb, b_scales, blocks_b * nkb);
    if (st) return st;
    auto run = [&](auto one, auto two, auto* out) -> int {
        if (pairs) {
            constexpr int smem = GP_STAGES * GP_STAGE_BYTES + 8 * 4096 + 1024;
            const int e = mx4_allow_smem(two, smem);
            if (e) return e;
            const int n = (int)(most < n_sm / 2 ? most : n_sm / 2);
            return rllm_launch_clusters(two, dim3(2 * n), dim3(GM_THREADS), smem, stream, dim3(2, 1, 1), maps, out, ldc, offsets, E, rows, N, K,
                                        glu, err);
        }
        constexpr int smem = GM_STAGES * GM_STAGE_BYTES + 8 * 4096 + 1024;
        const int e = mx4_allow_smem(one, smem);
        if (e) return e;
        return rllm_launch(one, dim3((unsigned)(most < n_sm ? most : n_sm)), dim3(GM_THREADS), smem, stream, maps.a, maps.b,
                           (const uint8_t*)a_scales, (const uint8_t*)b_scales, out, ldc, offsets, E, rows, N, K, ahead, glu, err);
    };
#define GM_RUN(TC, EPI) return run(gemm_mx4_kernel<TC, EPI>, gemm_mx4_pair_kernel<TC, EPI>, (TC*)C)
    if (epilogue == GM_EPI_ACCUM) GM_RUN(float, GM_EPI_ACCUM);
    if (epilogue == GM_EPI_GATED) { if (c_dtype == RLLM_F32) GM_RUN(float, GM_EPI_GATED); GM_RUN(bf16, GM_EPI_GATED); }
    if (epilogue == GM_EPI_STORE) { if (c_dtype == RLLM_F32) GM_RUN(float, GM_EPI_STORE); GM_RUN(bf16, GM_EPI_STORE); }
#undef GM_RUN
    return (int)cudaErrorInvalidValue;
}

// The whole product from rows x [rows of x, K] (float32 or bfloat16, ldx apart): they are quantised into `work` (codes, and from the next multiple
// of 1,024 bytes the scales), which rllm_gemm_mx4 then reads.  offsets, place, E, top_k as for rllm_mx4_quantize; `rows` sorted rows.
RLLM_API int rllm_mx4_product(const void* x, const int* offsets, const int* place, const void* w_codes, const void* w_scales, void* C,
                              void* work, int* err, long long ldx, long long ldc, int x_dtype, int c_dtype, int rows, int N, int K, int E,
                              int top_k, int epilogue, int pairs, int ahead, float glu_limit, float glu_alpha, float glu_shift, cudaStream_t stream) {
    if (rows <= 0 || N <= 0) return 0;
    unsigned char* scales = (unsigned char*)work + (((size_t)rows * (size_t)(K / 2) + 1023) & ~(size_t)1023);
    const int st = rllm_mx4_quantize(x, work, scales, offsets, place, ldx, x_dtype, rows, K, 0, E, top_k, stream);
    if (st) return st;
    return rllm_gemm_mx4(work, scales, w_codes, w_scales, C, c_dtype, ldc, offsets, E, rows, N, K, epilogue, pairs, ahead, glu_limit,
                         glu_alpha, glu_shift, err, stream);
}

TC_DEFINE_WAIT_CONTROLS(rllm_gemm_mx4)

RLLM_PACKED(rllm_mx4_product)
