// Block-scaled fp8 matmul on the tensor cores (sm_100a): tcgen05.mma kind::f8f6f4 with fp32 accumulators in tensor memory,
// operands straight from TMA-swizzled shared memory, and the fp32 scales applied block by block on the way out.
//
//   out[m,n] = sum_b xs[m,b] * ws[b,n/128] * ( sum_{k in block b} x[m,k] * w[k,n] ),   b = blocks of 128 k's
//
// The scales are arbitrary fp32 numbers, so a block's sum has to leave the accumulator before the next block's is added:
// every 128 k's the MMA warp starts a fresh accumulator (four instructions of K = 32) and the epilogue warps fold the finished one
// into fp32 registers, acc += part * (xs * ws), while the tensor cores work on the next.  Accumulators alternate in tensor memory.
//
// Two forms, by which operand lies on the accumulator's 128 lanes:
//   * rows on lanes (prefill): tile = 128 rows x 256 columns; xs * ws is one number per thread and block, since a thread holds
//     128 columns of one row and a weight block covers 128 columns.  Bound by the tensor pipe and the operand traffic from L2.
//   * columns on lanes (decode and few rows per expert): tile = 128 weight columns x 16..128 rows, so that few rows do not leave
//     the MMA's 128 lanes empty and the weights -- all of the traffic -- are read once.  A thread holds the rows of
//     one column; the rows' scales come from shared memory.  Bound by HBM.  When there are fewer tiles than SMs, a cluster of 2, 4
//     or 8 CTAs cuts K and sums its parts through distributed shared memory in rank order: one launch, no
//     workspace, the same bits every time.
//
// Weights [N,K] are the K-major operand form, [K,N] the MN-major one, which the instruction takes for 8-bit types; nothing is
// re-laid.  Experts: each CTA scans the row counts on the device into a table of row and tile starts, so the host never sees
// them; no tile crosses an expert.  Warps: 0 = TMA producer, 1 = MMA issuer and tensor-memory owner, the others = epilogue.
// Every wait is bounded and records a code in the device status word.
#include <algorithm>

#include "block_mm_common.cuh"

namespace qmm {
namespace {

// ROWS_ON_LANES: lanes = rows of x, columns = NT weight columns.  Else lanes = 128 weight columns, columns = NT rows of x.
template <bool ROWS_ON_LANES, int NT>
struct BmShape {
    static constexpr int L_BYTES = BM_LANES * BM_BK, C_BYTES = NT * BM_BK, STAGE = L_BYTES + C_BYTES;
    static constexpr int STAGES = ROWS_ON_LANES ? 4 : (NT <= 32 ? 9 : (NT <= 64 ? 8 : 6));
    static constexpr int NBUF = ROWS_ON_LANES ? 512 / NT : 4;
    static constexpr int TMEM_COLS = NBUF * NT;
    static constexpr int SETS = BM_EPI_WARPS / 4, COLS = NT / SETS;    // columns of a thread
    static constexpr int ROW_TILE = ROWS_ON_LANES ? BM_LANES : NT, COL_TILE = ROWS_ON_LANES ? NT : BM_LANES;
    static constexpr int TABLE_OFF = STAGES * STAGE;                   // row starts [E + 1], tile ends [E]
    static constexpr int FACT_OFF = TABLE_OFF + BM_TABLE_BYTES;
    static constexpr int BAR_OFF = FACT_OFF + BM_EPI_WARPS * COLS * 4;
    static constexpr int NUM_BARS = 2 * STAGES + 2 * NBUF;
    static constexpr int MISC_OFF = BAR_OFF + NUM_BARS * 8;
    static constexpr int TOTAL = MISC_OFF + 16 + 1024;
    static_assert(TOTAL <= 232448 && TMEM_COLS <= 512 && NT * 512 <= TABLE_OFF, "budgets of one CTA");
};

__device__ __forceinline__ void bm_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t local, uint32_t cta) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(cta));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}

template <bool ROWS_ON_LANES, int NT>
__global__ void __launch_bounds__(BM_THREADS, 1)
block_mm_tc_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const BmParams p, const uint32_t idesc) {
    using S = BmShape<ROWS_ON_LANES, NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *gen_base = smem_raw + (base - smem_u32(smem_raw));
    auto l_tile = [&](int s) { return base + s * S::STAGE; };
    auto c_tile = [&](int s) { return base + s * S::STAGE + S::L_BYTES; };
    auto bar_full = [&](int s) { return base + S::BAR_OFF + 8 * s; };
    auto bar_empty = [&](int s) { return base + S::BAR_OFF + 8 * (S::STAGES + s); };
    auto bar_acc_full = [&](int a) { return base + S::BAR_OFF + 8 * (2 * S::STAGES + a); };
    auto bar_acc_empty = [&](int a) { return base + S::BAR_OFF + 8 * (2 * S::STAGES + S::NBUF + a); };
    int *row_start = reinterpret_cast<int *>(gen_base + S::TABLE_OFF), *tile_end = row_start + p.E + 1;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(gen_base + S::MISC_OFF);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(gen_base + S::MISC_OFF + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
        for (int a = 0; a < S::NBUF; ++a) { mbar_init(bar_acc_full(a), 1); mbar_init(bar_acc_empty(a), BM_EPI_WARPS); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 1) tmem_alloc(smem_u32((const void *)tmem_slot), S::TMEM_COLS);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");   // everything below reads or writes global memory
    if (warp == 0) {
        fill_table<S::ROW_TILE>(p.counts, p.M, p.E, p.n_tiles, row_start, tile_end);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int tiles = tile_end[p.E - 1];
    // a cluster of `split` CTAs works on one tile, each on its part of the k blocks
    const int rank = (int)blockIdx.x % p.split, first = (int)blockIdx.x / p.split, step = (int)gridDim.x / p.split;
    const int kb0 = (int)((long long)p.nkb * rank / p.split), kb1 = (int)((long long)p.nkb * (rank + 1) / p.split);
    TileWalk<S::ROW_TILE, S::COL_TILE> walk{row_start, tile_end};

    int issued = 0;                                        // warp 0: stages filled; warp 1: blocks multiplied
    if (warp == 0) {
        int s = 0;
        uint32_t ph = 1;                                   // of bar_empty: the first round finds the stages free
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            int e, m0, rows, n0;
            walk.seek(tile, e, m0, rows, n0);
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!warp_wait(bar_empty(s), ph, abort_flag, 0x601u)) { ok = false; break; }
                if (elect_one()) {
                    mbar_expect_tx(bar_full(s), S::STAGE);
                    const int k = kb * BM_BK;
                    tma_load_2d(ROWS_ON_LANES ? l_tile(s) : c_tile(s), &tm_x, bar_full(s), k, m0);
                    const uint32_t wt = ROWS_ON_LANES ? c_tile(s) : l_tile(s);
                    if (p.w_nk) {
                        tma_load_3d(wt, &tm_w, bar_full(s), k, n0, e);
                    } else {
#pragma unroll
                        for (int h = 0; h < S::COL_TILE / 128; ++h) tma_load_3d(wt + h * 16384, &tm_w, bar_full(s), n0 + h * 128, k, e);
                    }
                }
                __syncwarp();
                ++issued;
                if (++s == S::STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        // K-major operands step 32 bytes along the row per K = 32, MN-major ones 32 rows of 128 bytes
        const uint32_t w_step = p.w_nk ? 32u : 4096u, w_lbo = p.w_nk ? 16u : 16384u;
        const uint64_t x_desc = smem_desc(ROWS_ON_LANES ? l_tile(0) : c_tile(0), 16, 1024), w_desc = smem_desc(ROWS_ON_LANES ? c_tile(0) : l_tile(0), w_lbo, 1024);
        int s = 0, a = 0;
        uint32_t ph = 0, aph = 1;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!warp_wait(bar_acc_empty(a), aph, abort_flag, 0x602u) || !warp_wait(bar_full(s), ph, abort_flag, 0x603u)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d = tmem_base + (uint32_t)(a * NT);
                const uint64_t xd = x_desc + (uint32_t)(s * (S::STAGE >> 4)), wd = w_desc + (uint32_t)(s * (S::STAGE >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint64_t xk = xd + (uint32_t)(kk * 2), wk = wd + kk * (w_step >> 4);
                        bm_mma(d, ROWS_ON_LANES ? xk : wk, ROWS_ON_LANES ? wk : xk, idesc, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(bar_empty(s));
                    tc_commit(bar_acc_full(a));
                }
                __syncwarp();
                ++issued;
                if (++s == S::STAGES) { s = 0; ph ^= 1u; }
                if (++a == S::NBUF) { a = 0; aph ^= 1u; }
            }
        }
    } else {
        const int ew = warp - 2, set = ew >> 2, q = warp & 3;
        const int ln = q * 32 + lane;                    // accumulator lane of this thread
        constexpr int CH = S::COLS < 16 ? S::COLS : 16, NCH = S::COLS / CH;
        float *fact = reinterpret_cast<float *>(gen_base + S::FACT_OFF) + ew * S::COLS;
        int it = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            int e, m0, rows, n0;
            walk.seek(tile, e, m0, rows, n0);
            // this thread's scales: of its row and its columns' weight block, or (lane by lane) of the set's rows
            const int nblk = ROWS_ON_LANES ? (n0 + set * S::COLS) / 128 : n0 / 128;
            const bool n_ok = nblk < p.nb;
            const float *wsp = p.ws + ((int64_t)e * p.nkb * p.nb + (n_ok ? (p.w_nk ? (int64_t)nblk * p.nkb : nblk) : 0));
            const int ws_step = p.w_nk ? 1 : p.nb;
            constexpr int RPL = ROWS_ON_LANES ? 1 : (S::COLS + 31) / 32;   // scales a lane fetches per block
            const float *xsp[RPL];
            bool x_ok[RPL];
#pragma unroll
            for (int i = 0; i < RPL; ++i) {
                const int r = ROWS_ON_LANES ? ln : set * S::COLS + lane + 32 * i;
                x_ok[i] = r < rows && (ROWS_ON_LANES || lane + 32 * i < S::COLS);
                xsp[i] = p.xs + (x_ok[i] ? (int64_t)(m0 + r) * p.nkb : 0);
            }
            // fetched two blocks ahead: a miss takes longer than a block
            float sw[2], sx[2][RPL];
            auto fetch = [&](int kb, int b) {
                sw[b] = n_ok && kb < kb1 ? __ldg(wsp + (int64_t)kb * ws_step) : 0.f;
#pragma unroll
                for (int i = 0; i < RPL; ++i) sx[b][i] = x_ok[i] && kb < kb1 ? __ldg(xsp[i] + kb) : 0.f;
            };
            fetch(kb0, 0);
            fetch(kb0 + 1, 1);
            uint64_t acc[S::COLS / 2];
#pragma unroll
            for (int i = 0; i < S::COLS / 2; ++i) acc[i] = 0ull;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int a = it % S::NBUF;
                uint64_t f2 = 0, fv[ROWS_ON_LANES ? 1 : S::COLS / 2];
                if constexpr (ROWS_ON_LANES) {
                    const float f = sx[0][0] * sw[0];
                    f2 = pack2(__float_as_uint(f), __float_as_uint(f));
                } else {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < RPL; ++i)
                        if (lane + 32 * i < S::COLS) fact[lane + 32 * i] = sx[0][i] * sw[0];
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < S::COLS / 4; ++i) {
                        const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(fact + 4 * i);
                        fv[2 * i] = t.x;
                        fv[2 * i + 1] = t.y;
                    }
                }
                sw[0] = sw[1];
#pragma unroll
                for (int i = 0; i < RPL; ++i) sx[0][i] = sx[1][i];
                fetch(kb + 2, 1);
                if (!warp_wait(bar_acc_full(a), (it / S::NBUF) & 1, abort_flag, 0x604u)) { ok = false; break; }
                tc_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * NT + set * S::COLS);
                uint32_t v[2][CH];
                bm_ld<CH>(taddr, v[0]);
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    bm_ld_wait<CH>(v[c & 1]);
                    if (c + 1 < NCH) bm_ld<CH>(taddr + (c + 1) * CH, v[(c + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < CH; i += 2)
                        fma2(acc[(c * CH + i) / 2], pack2(v[c & 1][i], v[c & 1][i + 1]), ROWS_ON_LANES ? f2 : fv[ROWS_ON_LANES ? 0 : (c * CH + i) / 2]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_acc_empty(a));
            }
            if (!ok) break;
            if constexpr (ROWS_ON_LANES) {
                const int nc = n0 + set * S::COLS;
                const int64_t at = (int64_t)(m0 + ln) * p.N + nc;
                if (ln >= rows) {
                    // a row behind the expert's last
                } else if (p.vec_out) {                    // N a multiple of 8, 16-byte aligned
                    uint8_t *o = (uint8_t *)p.out + at * (p.out_type == ET_F32 ? 4 : 2);
#pragma unroll
                    for (int g = 0; g < S::COLS / 8; ++g) {
                        if (nc + g * 8 >= p.N) break;
                        float f[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) unpack2(acc[g * 4 + i], f[2 * i], f[2 * i + 1]);
                        if (p.out_type == ET_F32) {
                            reinterpret_cast<float4 *>(o)[2 * g] = make_float4(f[0], f[1], f[2], f[3]);
                            reinterpret_cast<float4 *>(o)[2 * g + 1] = make_float4(f[4], f[5], f[6], f[7]);
                        } else {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (p.out_type == ET_BF16) { __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<uint32_t *>(&h); }
                                else { __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<uint32_t *>(&h); }
                            }
                            reinterpret_cast<uint4 *>(o)[g] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < S::COLS / 2; ++i) {
                        float f0, f1;
                        unpack2(acc[i], f0, f1);
                        if (nc + 2 * i < p.N) store_from_float(p.out, p.out_type, at + 2 * i, f0);
                        if (nc + 2 * i + 1 < p.N) store_from_float(p.out, p.out_type, at + 2 * i + 1, f1);
                    }
                }
            } else {
                const int n = n0 + ln;
                if (p.split > 1) {
                    // the ring is idle: this CTA's parts go there as [row][column], for every CTA of the cluster to read
                    float *red = reinterpret_cast<float *>(gen_base) + (set * S::COLS) * BM_LANES + ln;
#pragma unroll
                    for (int i = 0; i < S::COLS / 2; ++i) unpack2(acc[i], red[(2 * i) * BM_LANES], red[(2 * i + 1) * BM_LANES]);
                } else if (n < p.N) {
#pragma unroll
                    for (int i = 0; i < S::COLS; ++i) {
                        float f0, f1;
                        unpack2(acc[i / 2], f0, f1);
                        const int r = set * S::COLS + i;
                        if (r < rows) store_from_float(p.out, p.out_type, (int64_t)(m0 + r) * p.N + n, (i & 1) ? f1 : f0);
                    }
                }
            }
            __syncwarp();
        }
    }

    if constexpr (!ROWS_ON_LANES) {
        if (p.split > 1 && first < tiles) {               // one tile per cluster; the same for all of its CTAs
            bm_cluster_sync();
            if (warp >= 2) {
                int e, m0, rows, n0;
                TileWalk<S::ROW_TILE, S::COL_TILE> w2{row_start, tile_end};
                w2.seek(first, e, m0, rows, n0);
                // a warp sums a row: 4 columns a lane, all parts in flight, added in rank order
                for (int r = (warp - 2) * p.split + rank; r < rows; r += BM_EPI_WARPS * p.split) {
                    float4 part[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (c < p.split) part[c] = ld_cluster_f32x4(base + (uint32_t)(r * BM_LANES + lane * 4) * 4u, (uint32_t)c);
                    float4 v = part[0];
#pragma unroll
                    for (int c = 1; c < 8; ++c)
                        if (c < p.split) { v.x += part[c].x; v.y += part[c].y; v.z += part[c].z; v.w += part[c].w; }
                    const int n = n0 + lane * 4;
                    const int64_t at = (int64_t)(m0 + r) * p.N + n;
                    if (n < p.N) store_from_float(p.out, p.out_type, at, v.x);
                    if (n + 1 < p.N) store_from_float(p.out, p.out_type, at + 1, v.y);
                    if (n + 2 < p.N) store_from_float(p.out, p.out_type, at + 2, v.z);
                    if (n + 3 < p.N) store_from_float(p.out, p.out_type, at + 3, v.w);
                }
            }
            bm_cluster_sync();                            // a CTA's shared memory outlives the others' reads
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // a wait gave up: copies and products in flight end before the CTA's memory goes (each awaited with a limit)
        if (warp == 0 && lane == 0)
            for (int j = issued > S::STAGES ? issued - S::STAGES : 0; j < issued; ++j) bm_drain(bar_full(j % S::STAGES), (j / S::STAGES) & 1);
        if (warp == 1 && lane == 0)
            for (int j = issued > S::NBUF ? issued - S::NBUF : 0; j < issued; ++j) bm_drain(bar_acc_full(j % S::NBUF), (j / S::NBUF) & 1);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, S::TMEM_COLS);
    }
}

template <bool ROWS_ON_LANES, int NT> cudaError_t launch_form(const BlockMmArgs &a, int split, cudaStream_t s) {
    using S = BmShape<ROWS_ON_LANES, NT>;
    const int E = a.experts > 0 ? (int)a.experts : 1;
    CUtensorMap tx, tw;
    bool ok = make_map(&tx, a.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.K, a.M, a.K, BM_BK, S::ROW_TILE, CU_TENSOR_MAP_SWIZZLE_128B);
    ok = ok && (a.w_nk ? make_map3(&tw, a.w, a.K, a.N, E, BM_BK, S::COL_TILE) : make_map3(&tw, a.w, a.N, a.K, E, 128, BM_BK));
    if (!ok) return cudaErrorInvalidValue;
    BmParams p{};
    p.xs = a.xs; p.ws = a.ws; p.counts = a.experts > 0 ? a.group_rows : nullptr; p.out = a.out; p.out_type = a.out_type;
    p.vec_out = a.N % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
    p.M = (int)a.M; p.N = (int)a.N; p.nkb = (int)((a.K + BM_BK - 1) / BM_BK); p.nb = (int)((a.N + 127) / 128); p.E = E;
    p.n_tiles = (int)((a.N + S::COL_TILE - 1) / S::COL_TILE); p.w_nk = a.w_nk; p.split = split;
    const int x_fmt = a.x_type == ET_E5M2, w_fmt = a.w_type == ET_E5M2, w_mn = a.w_nk ? 0 : 1;
    const uint32_t idesc = ROWS_ON_LANES ? bm_idesc(x_fmt, w_fmt, 0, w_mn, BM_LANES, NT) : bm_idesc(w_fmt, x_fmt, w_mn, 0, BM_LANES, NT);
    // tiles: each expert with rows adds at most one partly filled row tile
    const int64_t full = (a.M + S::ROW_TILE - 1) / S::ROW_TILE, most = a.experts > 0 ? std::min<int64_t>(a.M, full + E - 1) : full;
    const int64_t tiles = most * p.n_tiles;
    const int64_t grid = split > 1 ? tiles * split : std::min<int64_t>(tiles, sm_count());
    cudaError_t e = allow_smem<block_mm_tc_kernel<ROWS_ON_LANES, NT>>(S::TOTAL);
    if (e != cudaSuccess) return e;
    e = launch_chained(block_mm_tc_kernel<ROWS_ON_LANES, NT>, (unsigned)grid, BM_THREADS, S::TOTAL, (unsigned)split, s, tx, tw, p, idesc);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace

bool block_mm_tc_supported(const BlockMmArgs &a) {
    auto al16 = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    if (!al16(a.x) || !al16(a.w) || a.K % 16 != 0 || (!a.w_nk && a.N % 16 != 0)) return false;
    // tile numbers are 32-bit
    return (a.M / 16 + a.experts + 1) * ((a.N + 127) / 128) < (1LL << 30);
}

cudaError_t launch_block_mm_tc(const BlockMmArgs &a, cudaStream_t s) {
    const int64_t rows = a.experts > 0 ? (a.M + a.experts - 1) / a.experts : a.M;   // of an expert, on average
    if (rows > 128) return getenv("BM_SINGLE") ? launch_form<true, 256>(a, 1, s) : launch_block_mm_pair(a, s);
    const int nt = rows <= 8 ? 16 : (rows <= 24 ? 32 : (rows <= 56 ? 64 : 128));
    const int64_t nkb = (a.K + BM_BK - 1) / BM_BK, cols = (a.N + 127) / 128, full = (a.M + nt - 1) / nt;
    const int64_t tiles = (a.experts > 0 ? std::min<int64_t>(a.M, full + a.experts - 1) : full) * cols;
    int split = 1;
    while (split < 8 && tiles * split * 2 <= sm_count() && split * 4 <= nkb) split *= 2;
    switch (nt) {
        case 16: return launch_form<false, 16>(a, split, s);
        case 32: return launch_form<false, 32>(a, split, s);
        case 64: return launch_form<false, 64>(a, split, s);
        default: return launch_form<false, 128>(a, split, s);
    }
}

unsigned int block_mm_device_status() {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tc_status, sizeof(v)) != cudaSuccess) return 0xFFFFFFFFu;
    return v ? v : block_mm_pair_device_status();
}
void block_mm_device_status_reset() {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_tc_status, &z, sizeof(z));
    block_mm_pair_device_status_reset();
}

}  // namespace qmm
