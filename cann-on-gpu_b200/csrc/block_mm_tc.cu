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

#include "launch_utils.h"
#include "tc_common.cuh"

namespace qmm {
namespace {

constexpr int BM_LANES = 128, BM_BK = 128, BM_EPI_WARPS = 8, BM_THREADS = 64 + BM_EPI_WARPS * 32;

struct BmParams {
    const float *xs, *ws;
    const int64_t *counts;      // [E] on the device, or null
    void *out;
    int out_type, vec_out;
    int M, N, nkb, nb, E;       // E >= 1 (dense: 1)
    int n_tiles, w_nk, split;
};

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
    static constexpr int FACT_OFF = TABLE_OFF + (2 * BLOCK_MM_MAX_EXPERTS + 4) * 4;
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
// D fp32, A / B formats (0 = e4m3, 1 = e5m2), A and B MN-major flags.
constexpr uint32_t bm_idesc(int a_fmt, int b_fmt, int a_mn, int b_mn, int m, int n) {
    return (1u << 4) | ((uint32_t)a_fmt << 7) | ((uint32_t)b_fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(tm), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// tcgen05.ld of 8 or 16 columns without the wait; the wait takes the registers so that no use moves in front of it.
template <int N> __device__ __forceinline__ void bm_ld(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                       "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
template <int N> __device__ __forceinline__ void bm_ld_wait(uint32_t (&r)[N]) {
    if constexpr (N == 16)
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                       "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
    else
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]) :: "memory");
}
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    lo = __uint_as_float(a);
    hi = __uint_as_float(b);
}
// Two fp32 fused multiply-adds in one instruction.
__device__ __forceinline__ void fma2(uint64_t &acc, uint64_t a, uint64_t b) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b)); }

__device__ __forceinline__ void bm_drain(uint32_t bar, uint32_t parity) {
    const unsigned long long t0 = global_ns();
    while (!mbar_try_wait(bar, parity) && global_ns() - t0 < 50000000ull) {}
}

__device__ __forceinline__ void bm_cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t local, uint32_t cta) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// Tile t in ascending t: expert, first row and rows, first column.
template <int ROW_TILE, int COL_TILE>
struct TileWalk {
    const int *row_start, *tile_end;
    int e = 0;
    __device__ __forceinline__ void seek(int tile, int &expert, int &m0, int &rows, int &n0) {
        while (tile >= tile_end[e]) ++e;
        const int local = tile - (e ? tile_end[e - 1] : 0), r0 = row_start[e], r1 = row_start[e + 1];
        const int mt = (r1 - r0 + ROW_TILE - 1) / ROW_TILE;
        const int nt = local / mt;
        m0 = r0 + (local - nt * mt) * ROW_TILE;
        rows = r1 - m0 < ROW_TILE ? r1 - m0 : ROW_TILE;
        n0 = nt * COL_TILE;
        expert = e;
    }
};

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
        if (!p.counts) {
            if (lane == 0) { row_start[0] = 0; row_start[1] = p.M; tile_end[0] = (p.M + S::ROW_TILE - 1) / S::ROW_TILE * p.n_tiles; }
        } else {
            // counts below 0 count as 0, and rows end at M
            int rows = 0, tiles = 0;
            for (int e0 = 0; e0 < p.E; e0 += 32) {
                const int e = e0 + lane;
                long long c = e < p.E ? __ldg((const long long *)p.counts + e) : 0;
                c = c < 0 ? 0 : (c > p.M ? p.M : c);
                long long end = c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long v = __shfl_up_sync(0xffffffffu, end, o);
                    if (lane >= o) end += v;
                }
                const long long lo64 = rows + end - c, hi64 = rows + end;
                const int lo = (int)(lo64 < p.M ? lo64 : p.M), hi = (int)(hi64 < p.M ? hi64 : p.M);
                int t = (hi - lo + S::ROW_TILE - 1) / S::ROW_TILE * p.n_tiles;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, t, o);
                    if (lane >= o) t += v;
                }
                if (e < p.E) { row_start[e] = lo; tile_end[e] = tiles + t; if (e == p.E - 1) row_start[p.E] = hi; }
                rows = __shfl_sync(0xffffffffu, hi, 31);
                tiles += __shfl_sync(0xffffffffu, t, 31);
            }
        }
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
        if (lane == 0) {
            int &it = issued;
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += step) {
                int e, m0, rows, n0;
                walk.seek(tile, e, m0, rows, n0);
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % S::STAGES;
                    if (it >= S::STAGES && !mbar_wait(bar_empty(s), ((it / S::STAGES) - 1) & 1, abort_flag, 0x601u)) { ok = false; break; }
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
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // K-major operands step 32 bytes along the row per K = 32, MN-major ones 32 rows of 128 bytes
            const uint32_t w_step = p.w_nk ? 32u : 4096u, w_lbo = p.w_nk ? 16u : 16384u;
            int &it = issued;
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += step) {
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % S::STAGES, a = it % S::NBUF;
                    if (it >= S::NBUF && !mbar_wait(bar_acc_empty(a), ((it / S::NBUF) - 1) & 1, abort_flag, 0x602u)) { ok = false; break; }
                    if (!mbar_wait(bar_full(s), (it / S::STAGES) & 1, abort_flag, 0x603u)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t d = tmem_base + (uint32_t)(a * NT);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint64_t xd = smem_desc((ROWS_ON_LANES ? l_tile(s) : c_tile(s)) + kk * 32, 16, 1024);
                        const uint64_t wd = smem_desc((ROWS_ON_LANES ? c_tile(s) : l_tile(s)) + kk * w_step, w_lbo, 1024);
                        bm_mma(d, ROWS_ON_LANES ? xd : wd, ROWS_ON_LANES ? wd : xd, idesc, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(bar_empty(s));
                    tc_commit(bar_acc_full(a));
                }
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
            float sw = 0.f, sx[RPL];
            auto fetch = [&](int kb) {
                sw = n_ok && kb < kb1 ? __ldg(wsp + (int64_t)kb * ws_step) : 0.f;
#pragma unroll
                for (int i = 0; i < RPL; ++i) sx[i] = x_ok[i] && kb < kb1 ? __ldg(xsp[i] + kb) : 0.f;
            };
            fetch(kb0);
            uint64_t acc[S::COLS / 2];
#pragma unroll
            for (int i = 0; i < S::COLS / 2; ++i) acc[i] = 0ull;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int a = it % S::NBUF;
                uint64_t f2 = 0;
                if constexpr (ROWS_ON_LANES) {
                    const float f = sx[0] * sw;
                    f2 = pack2(__float_as_uint(f), __float_as_uint(f));
                } else {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < RPL; ++i)
                        if (lane + 32 * i < S::COLS) fact[lane + 32 * i] = sx[i] * sw;
                    __syncwarp();
                }
                fetch(kb + 1);
                // (a vote, so that a wait that gave up takes the whole warp along)
                if (!__all_sync(0xffffffffu, mbar_wait(bar_acc_full(a), (it / S::NBUF) & 1, abort_flag, 0x604u))) { ok = false; break; }
                tc_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * NT + set * S::COLS);
                uint32_t v[2][CH];
                bm_ld<CH>(taddr, v[0]);
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    bm_ld_wait<CH>(v[c & 1]);
                    if (c + 1 < NCH) bm_ld<CH>(taddr + (c + 1) * CH, v[(c + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < CH; i += 4) {
                        uint64_t f0 = f2, f1 = f2;
                        if constexpr (!ROWS_ON_LANES) {
                            const ulonglong2 fv = *reinterpret_cast<const ulonglong2 *>(fact + c * CH + i);
                            f0 = fv.x;
                            f1 = fv.y;
                        }
                        fma2(acc[(c * CH + i) / 2], pack2(v[c & 1][i], v[c & 1][i + 1]), f0);
                        fma2(acc[(c * CH + i) / 2 + 1], pack2(v[c & 1][i + 2], v[c & 1][i + 3]), f1);
                    }
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
                const int t = threadIdx.x - 64, ln = t & 127, n = n0 + ln;
                for (int r = (t >> 7) * p.split + rank; r < rows; r += S::SETS * p.split) {
                    float v = 0.f;
                    for (int c = 0; c < p.split; ++c) v += ld_cluster_f32(base + (uint32_t)(r * BM_LANES + ln) * 4u, (uint32_t)c);
                    if (n < p.N) store_from_float(p.out, p.out_type, (int64_t)(m0 + r) * p.N + n, v);
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

// 3-D map of E matrices of `rows` rows of `cols` bytes.
bool make_map3(CUtensorMap *tm, const void *ptr, uint64_t cols, uint64_t rows, uint64_t E, uint32_t box_cols, uint32_t box_rows) {
    EncodeFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {cols, rows, E}, strides[2] = {cols, cols * rows};
    cuuint32_t box[3] = {box_cols, box_rows, 1}, estr[3] = {1, 1, 1};
    return fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
    if (rows > 128) return launch_form<true, 256>(a, 1, s);
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
    return v;
}
void block_mm_device_status_reset() {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_tc_status, &z, sizeof(z));
}

}  // namespace qmm
