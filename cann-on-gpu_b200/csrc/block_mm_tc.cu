// Block-scaled fp8 matmul on the tensor cores for few rows (decode, or few rows per expert).
//
//   out[m,n] = sum_b xs[m,b] * ws[b,n/128] * ( sum_{k in block b} x[m,k] * w[k,n] ),   b = blocks of 128 k's
//
// The 128 lanes of the accumulator are weight columns and its 16, 32 or 64 columns are rows of x, so that few rows do not leave
// the tensor core's lanes empty and the weights -- nearly all of the traffic -- are read once.  The kernel is bound by HBM as long as a
// block of 16 KB of weights passes an SM in under 700 cycles, and what has to fit in there is not the arithmetic but the
// hand-overs (a ready barrier costs some 100 cycles to pass, four products 200 to issue), so they move two blocks at a time.
//
// The scales are arbitrary fp32 numbers, so a block's sum leaves tensor memory before the next block's is added: the
// epilogue warps fold it into fp32 registers, acc += part * (xs[row] * ws), a thread holding the rows of one column.
//
// Weights [N,K] are the K-major operand form, [K,N] the MN-major one, which the instruction takes for 8-bit types; nothing is
// re-laid.  Experts: each CTA scans the row counts on the device into a table of row and tile starts, so the host never sees
// them; no tile crosses an expert.  When there are fewer tiles than SMs, a cluster of 2, 4 or 8 CTAs cuts K and sums its
// parts through distributed shared memory in rank order: one launch, no workspace, the same bits every time.
//
// Warps: 0 = TMA producer, 1 = MMA issuer and tensor-memory owner, 2 = scales, 4-11 = epilogue (two sets of four,
// half of the rows each).  Every wait is bounded and records a code in the device status word.
#include <algorithm>
#include <cmath>

#include "block_mm_common.cuh"

namespace qmm {
namespace {

constexpr int BT_EPI = 8, BT_THREADS = 128 + BT_EPI * 32, BT_SLOTS = 8, BT_AHEAD = 4;

// NT rows of x per tile.  A group is two blocks of 128 k's.
template <int NT>
struct BtShape {
    static constexpr int W_BYTES = BM_LANES * BM_BK, X_BYTES = NT * BM_BK, STAGE = 2 * (W_BYTES + X_BYTES);
    static constexpr int STAGES = NT <= 32 ? 5 : 4;
    static constexpr int NBUF = 2, TMEM_COLS = 2 * NBUF * NT;          // accumulators: NBUF groups of two
    static constexpr int COLS = NT / 2;                                // rows of x of a thread
    static constexpr int TABLE_OFF = STAGES * STAGE;
    static constexpr int SC_OFF = TABLE_OFF + BM_TABLE_BYTES;          // slots of two blocks: NT row scales, the weight's and 3 unused
    static constexpr int SC_BLOCK = (NT + 4) * 4, SC_SLOT = 2 * SC_BLOCK;
    static constexpr int BAR_OFF = SC_OFF + BT_SLOTS * SC_SLOT;
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
// The first `rows` of a thread's sums to one column of out.
template <int T, int PAIRS, typename E>
__device__ __forceinline__ void store_column(const uint64_t (&acc)[PAIRS], E *o, int rows, int N) {
#pragma unroll
    for (int i = 0; i < 2 * PAIRS; i += 2) {
        float f0, f1;
        E e0, e1;
        unpack2(acc[i / 2], f0, f1);
        if constexpr (T == ET_F32) {
            e0 = f0; e1 = f1;
        } else {
            uint32_t h;
            if constexpr (T == ET_BF16) { __nv_bfloat162 b = __floats2bfloat162_rn(f0, f1); h = *reinterpret_cast<uint32_t *>(&b); }
            else { __half2 b = __floats2half2_rn(f0, f1); h = *reinterpret_cast<uint32_t *>(&b); }
            e0 = (E)h; e1 = (E)(h >> 16);
        }
        if (i < rows) *o = e0;
        o += N;
        if (i + 1 < rows) *o = e1;
        o += N;
    }
}
template <int NT>
__global__ void __launch_bounds__(BT_THREADS, 1)
block_mm_tc_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const BmParams p, const uint32_t idesc) {
    using S = BtShape<NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *gen_base = smem_raw + (base - smem_u32(smem_raw));
    auto w_tile = [&](int s, int b) { return base + s * S::STAGE + b * S::W_BYTES; };
    auto x_tile = [&](int s, int b) { return base + s * S::STAGE + 2 * S::W_BYTES + b * S::X_BYTES; };
    auto bar_full = [&](int s) { return base + S::BAR_OFF + 8 * s; };
    auto bar_empty = [&](int s) { return base + S::BAR_OFF + 8 * (S::STAGES + s); };
    auto bar_acc_full = [&](int a) { return base + S::BAR_OFF + 8 * (2 * S::STAGES + a); };     // products and scales of a group
    auto bar_acc_empty = [&](int a) { return base + S::BAR_OFF + 8 * (2 * S::STAGES + S::NBUF + a); };
    int *row_start = reinterpret_cast<int *>(gen_base + S::TABLE_OFF), *tile_end = row_start + p.E + 1;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(gen_base + S::MISC_OFF);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(gen_base + S::MISC_OFF + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
        for (int a = 0; a < S::NBUF; ++a) { mbar_init(bar_acc_full(a), 2); mbar_init(bar_acc_empty(a), BT_EPI); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 1) tmem_alloc(smem_u32((const void *)tmem_slot), S::TMEM_COLS);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");   // everything below reads or writes global memory
    if (warp == 0) fill_table<NT>(p.counts, p.M, p.E, p.n_tiles, row_start, tile_end);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int tiles = tile_end[p.E - 1];
    // a cluster of `split` CTAs works on one tile, each on its part of the groups
    const int rank = (int)blockIdx.x % p.split, first = (int)blockIdx.x / p.split, step = (int)gridDim.x / p.split;
    const int groups = (p.nkb + 1) / 2;
    const int g0 = (int)((long long)groups * rank / p.split), g1 = (int)((long long)groups * (rank + 1) / p.split);
    TileWalk<NT, BM_LANES> walk{row_start, tile_end};
    int issued = 0;                                       // warp 0: stages filled; warp 1: groups multiplied

    if (warp < 4) {
        // 384 threads x 168 registers at launch = 128 x 56 + 256 x 224
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            int s = 0;
            uint32_t ph = 1;                              // of bar_empty: the first round finds the stages free
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += step) {
                int e, m0, rows, n0;
                walk.seek(tile, e, m0, rows, n0);
                for (int g = g0; g < g1; ++g) {
                    if (!warp_wait(bar_empty(s), ph, abort_flag, 0x601u)) { ok = false; break; }
                    if (elect_one()) {
                        // (a second block behind K arrives as zeros and is not folded)
                        mbar_expect_tx(bar_full(s), S::STAGE);
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const int k = (2 * g + b) * BM_BK;
                            tma_load_3d(w_tile(s, b), &tm_w, bar_full(s), p.w_nk ? k : n0, p.w_nk ? n0 : k, e);
                            tma_load_2d(x_tile(s, b), &tm_x, bar_full(s), k, m0);
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
            const uint64_t x_desc = smem_desc(x_tile(0, 0), 16, 1024), w_desc = smem_desc(w_tile(0, 0), w_lbo, 1024);
            int s = 0, a = 0;
            uint32_t ph = 0, aph = 1;
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += step) {
                for (int g = g0; g < g1; ++g) {
                    if (!warp_wait(bar_acc_empty(a), aph, abort_flag, 0x602u) || !warp_wait(bar_full(s), ph, abort_flag, 0x603u)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t xd = x_desc + (uint32_t)(s * (S::STAGE >> 4)), wd = w_desc + (uint32_t)(s * (S::STAGE >> 4));
                    if (elect_one()) {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                bm_mma(tmem_base + (uint32_t)((2 * a + b) * NT), wd + (uint32_t)(b * (S::W_BYTES >> 4)) + kk * (w_step >> 4),
                                       xd + (uint32_t)(b * (S::X_BYTES >> 4) + kk * 2), idesc, kk > 0 ? 1u : 0u);
                        tc_commit(bar_acc_full(a));
                        tc_commit(bar_empty(s));
                    }
                    __syncwarp();
                    ++issued;
                    if (++s == S::STAGES) { s = 0; ph ^= 1u; }
                    a ^= 1;
                    if (a == 0) aph ^= 1u;
                }
            }
        } else if (warp == 2) {
            // scales: the copies run BT_AHEAD groups in front of the reports.  A report for group i waits for group i - 2
            // to be complete, by when group i - 4 has been folded and its slot of 8 is free for group i + 4.
            TileWalk<NT, BM_LANES> ahead{row_start, tile_end};
            constexpr int RPL = (NT + 31) / 32;
            int atile = first, ag = g0, slot = 0, rows = 0;
            const float *xsp = p.xs, *wsp = p.ws;
            const int ws_step = p.w_nk ? 1 : p.nb;
            auto copy_next = [&] {                        // one commit group per call, empty behind the last tile
                if (atile < tiles && g0 < g1) {
                    if (ag == g0) {
                        int e, m0, n0;
                        ahead.seek(atile, e, m0, rows, n0);
                        xsp = p.xs + (int64_t)(m0 + lane) * p.nkb;
                        wsp = p.ws + (int64_t)e * p.nkb * p.nb + (p.w_nk ? (int64_t)(n0 / 128) * p.nkb : n0 / 128);
                    }
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int kb = 2 * ag + b;
                        const uint32_t dst = base + S::SC_OFF + (uint32_t)(slot * S::SC_SLOT + b * S::SC_BLOCK);
                        if (kb >= p.nkb) break;
#pragma unroll
                        for (int i = 0; i < RPL; ++i)
                            if (lane + 32 * i < rows) cp_async4(dst + (lane + 32 * i) * 4, xsp + (int64_t)(32 * i) * p.nkb + kb);
                        if (lane == 0) cp_async4(dst + NT * 4, wsp + (int64_t)kb * ws_step);
                    }
                    if (++ag == g1) { ag = g0; atile += step; }
                    slot = (slot + 1) & (BT_SLOTS - 1);
                }
                cp_async_commit();
            };
            for (int i = 0; i < BT_AHEAD; ++i) copy_next();
            int a = 0;
            uint32_t ph = 1;                              // of the accumulator's previous use
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += step) {
                for (int g = g0; g < g1; ++g) {
                    if (!warp_wait(bar_acc_full(a), ph, abort_flag, 0x605u)) { ok = false; break; }
                    copy_next();
                    cp_async_wait<BT_AHEAD>();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_acc_full(a));
                    a ^= 1;
                    if (a == 0) ph ^= 1u;
                }
            }
            cp_async_wait<0>();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int ew = warp - 4, set = ew >> 2, q = warp & 3;
        const int ln = q * 32 + lane;                     // accumulator lane of this thread
        constexpr int CH = S::COLS < 32 ? S::COLS : 32, NCH = S::COLS / CH;
        const uint32_t tm_lane = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(set * S::COLS);
        int a = 0, slot = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            uint64_t acc[S::COLS / 2];
#pragma unroll
            for (int i = 0; i < S::COLS / 2; ++i) acc[i] = 0ull;
            for (int g = g0; g < g1; ++g) {
                if (!warp_wait(bar_acc_full(a), ph, abort_flag, 0x604u)) { ok = false; break; }
                tc_fence_after();
                const uint32_t taddr = tm_lane + (uint32_t)(2 * a * NT);
                const float *sc = reinterpret_cast<const float *>(gen_base + S::SC_OFF + slot * S::SC_SLOT);
                const bool two = 2 * g + 1 < p.nkb;
                uint32_t v[2][CH];
                bm_ld<CH>(taddr, v[0]);
#pragma unroll
                for (int c = 0; c < 2 * NCH; ++c) {       // NCH pieces of each of the two blocks
                    const int b = c / NCH, i0 = (c % NCH) * CH;
                    const float sw = sc[b * (S::SC_BLOCK / 4) + NT];
                    const uint64_t sw2 = pack2(__float_as_uint(sw), __float_as_uint(sw));
                    const float *sx = sc + b * (S::SC_BLOCK / 4) + set * S::COLS + i0;
                    uint64_t f[CH / 2];
#pragma unroll
                    for (int i = 0; i < CH / 2; i += 2) {
                        const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(sx + 2 * i);
                        f[i] = mul2(t.x, sw2);
                        f[i + 1] = mul2(t.y, sw2);
                    }
                    bm_ld_wait<CH>(v[c & 1]);
                    if (c + 1 < 2 * NCH) {
                        bm_ld<CH>(taddr + (uint32_t)((c + 1) / NCH * NT + (c + 1) % NCH * CH), v[(c + 1) & 1]);
                    } else {                              // all of it is in registers: the accumulators are free
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar_acc_empty(a));
                    }
                    if (b == 0 || two) {
#pragma unroll
                        for (int i = 0; i < CH; i += 2) fma2(acc[(i0 + i) / 2], pack2(v[c & 1][i], v[c & 1][i + 1]), f[i / 2]);
                    }
                }
                slot = (slot + 1) & (BT_SLOTS - 1);
                a ^= 1;
                if (a == 0) ph ^= 1u;
            }
            if (!ok) break;
            if (p.split > 1) {
                // the ring is idle: this CTA's parts go there as [row][column], for every CTA of the cluster to read
                float *red = reinterpret_cast<float *>(gen_base) + (set * S::COLS) * BM_LANES + ln;
#pragma unroll
                for (int i = 0; i < S::COLS / 2; ++i) unpack2(acc[i], red[(2 * i) * BM_LANES], red[(2 * i + 1) * BM_LANES]);
            } else {
                int e, m0, rows, n0;
                walk.seek(tile, e, m0, rows, n0);
                const int n = n0 + ln, r0 = set * S::COLS;
                if (n < p.N) {
                    const int64_t at = (int64_t)(m0 + r0) * p.N + n;
                    if (p.out_type == ET_BF16) store_column<ET_BF16>(acc, (uint16_t *)p.out + at, rows - r0, p.N);
                    else if (p.out_type == ET_F16) store_column<ET_F16>(acc, (uint16_t *)p.out + at, rows - r0, p.N);
                    else store_column<ET_F32>(acc, (float *)p.out + at, rows - r0, p.N);
                }
                __syncwarp();
            }
        }
    }

    if (p.split > 1 && first < tiles) {                   // one tile per cluster; the same for all of its CTAs
        bm_cluster_sync();
        if (warp >= 4) {
            int e, m0, rows, n0;
            TileWalk<NT, BM_LANES> w2{row_start, tile_end};
            w2.seek(first, e, m0, rows, n0);
            // a warp sums a row: 4 columns a lane, all parts in flight, added in rank order
            for (int r = (warp - 4) * p.split + rank; r < rows; r += BT_EPI * p.split) {
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
                if (p.out_type == ET_BF16) store_quad<ET_BF16>(p.out, p.vec_out, at, p.N - n, v);
                else if (p.out_type == ET_F16) store_quad<ET_F16>(p.out, p.vec_out, at, p.N - n, v);
                else store_quad<ET_F32>(p.out, p.vec_out, at, p.N - n, v);
            }
        }
        bm_cluster_sync();                                // a CTA's shared memory outlives the others' reads
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

template <int NT> cudaError_t launch_form(const BlockMmArgs &a, int split, cudaStream_t s) {
    using S = BtShape<NT>;
    const int E = a.experts > 0 ? (int)a.experts : 1;
    CUtensorMap tx, tw;
    bool ok = make_map(&tx, a.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.K, a.M, a.K, BM_BK, NT, CU_TENSOR_MAP_SWIZZLE_128B);
    ok = ok && (a.w_nk ? make_map3(&tw, a.w, a.K, a.N, E, BM_BK, BM_LANES) : make_map3(&tw, a.w, a.N, a.K, E, BM_LANES, BM_BK));
    if (!ok) return cudaErrorInvalidValue;
    BmParams p{};
    p.xs = a.xs; p.ws = a.ws; p.counts = a.experts > 0 ? a.group_rows : nullptr; p.out = a.out; p.out_type = a.out_type;
    p.M = (int)a.M; p.N = (int)a.N; p.nkb = (int)((a.K + BM_BK - 1) / BM_BK); p.nb = (int)((a.N + 127) / 128); p.E = E;
    p.vec_out = a.N % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
    p.n_tiles = (int)((a.N + BM_LANES - 1) / BM_LANES); p.w_nk = a.w_nk; p.split = split;
    const uint32_t idesc = bm_idesc(a.w_type == ET_E5M2, a.x_type == ET_E5M2, a.w_nk ? 0 : 1, 0, BM_LANES, NT);
    // tiles: each expert with rows adds at most one partly filled row tile
    const int64_t full = (a.M + NT - 1) / NT, most = a.experts > 0 ? std::min<int64_t>(a.M, full + E - 1) : full;
    const int64_t tiles = most * p.n_tiles;
    const int64_t grid = split > 1 ? tiles * split : std::min<int64_t>(tiles, sm_count());
    cudaError_t e = allow_smem<block_mm_tc_kernel<NT>>(S::TOTAL);
    if (e != cudaSuccess) return e;
    if (!has_regs<block_mm_tc_kernel<NT>>(168)) return cudaErrorInvalidConfiguration;
    return launch_chained(block_mm_tc_kernel<NT>, (unsigned)grid, BT_THREADS, S::TOTAL, (unsigned)split, s, tx, tw, p, idesc);
}

}  // namespace
bool block_mm_tc_supported(const BlockMmArgs &a) {
    auto al16 = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    if (!al16(a.x) || !al16(a.w) || a.K % 16 != 0 || (!a.w_nk && a.N % 16 != 0)) return false;
    // tile numbers are 32-bit
    return (a.M / 16 + a.experts + 1) * ((a.N + 127) / 128) < (1LL << 30);
}

// The form with the least estimated time (us): a fixed part, and the longer of two, the weights from HBM or the rounds of tiles
// over the SMs, with some of the shorter.  A round is the measured time of a step of K -- 0.36, 0.40 and 0.50 per group of two
// blocks with 16, 32 and 64 rows a tile, 0.41 per block and pair of CTAs with 256 x 256 tiles -- and of a tile's stores.
// Measured with 16 / 32 / 64 rows a tile / pairs: 64 x 4096 x 14336 27.7 / 17.8 / 14.5 / 19.0, 128 x 4096 x 14336 - / 29.2 / 20.7 / 19.8,
// 256 x 4096 x 4096 - / - / 12.2 / 17.4, 64 experts of 2048 x 2816 with 4 rows each 54 / 54 / 56 / 76, with 32 rows 85 / 69 / 67 / 88, with 128
// rows - / 157 / 120 / 110.  Tiles of 128 rows on one CTA were the fastest nowhere (21.7 and 16.9 on the second and third).
// The rows of an expert are not known here: their mean stands in, with half a tile more per expert.
cudaError_t launch_block_mm_tc(const BlockMmArgs &a, cudaStream_t s) {
    const int64_t nkb = (a.K + BM_BK - 1) / BM_BK, groups = (nkb + 1) / 2, sms = sm_count();
    const double experts = a.experts > 0 ? (double)std::min(a.experts, a.M) : 1.0, mean = (double)a.M / experts;
    const double hbm = experts * (double)a.K * (double)a.N / 6.2e6;
    auto rounds = [&](int tile_rows, int tile_cols, double slots) {
        const double per = a.experts > 0 ? std::max(1.0, mean / tile_rows + 0.5) : std::ceil(mean / tile_rows);
        return std::ceil(experts * per * (double)((a.N + tile_cols - 1) / tile_cols) / slots);
    };
    auto time = [&](double fixed, double sm) { return fixed + std::max(hbm, sm) + 0.15 * std::min(hbm, sm); };
    // the most tiles there can be, whatever the experts' rows: a cluster that cuts K has one tile
    auto most = [&](int tile_rows, int tile_cols) {
        const int64_t full = (a.M + tile_rows - 1) / tile_rows;
        return (a.experts > 0 ? std::min<int64_t>(a.M, full + a.experts - 1) : full) * ((a.N + tile_cols - 1) / tile_cols);
    };
    // clusters of 2, 4 and 8 CTAs, one CTA per SM, that run at once: 74, 33 and 15 with 148 SMs (none crosses a GPC)
    auto clusters = [&](int ctas) { return ctas == 1 ? sms : (ctas == 2 ? sms / 2 : (ctas == 4 ? sms * 33 / 148 : sms * 15 / 148)); };
    int best_nt = 0, best_split = 1;
    double best = time(6.2, rounds(256, 256, (double)(sms / 2)) * ((double)nkb * 0.41 + 1.3));
    for (int split = 2; split <= 4; split *= 2) {
        if (most(256, 256) > clusters(2 * split) || split * 8 > nkb) break;
        const double t = time(split == 2 ? 7.2 : 9.2, (double)((nkb + split - 1) / split) * 0.41 + 1.3);
        if (t < best) { best = t; best_split = split; }
    }
    const int nts[3] = {16, 32, 64};
    const double step_us[3] = {0.36, 0.40, 0.50};
    for (int i = 0; i < 3; ++i) {
        int split = 1;
        while (split < 8 && most(nts[i], BM_LANES) <= clusters(2 * split) && split * 4 <= groups) split *= 2;
        // (where K is cut all tiles run at once)
        const double r = split > 1 ? 1.0 : rounds(nts[i], BM_LANES, (double)sms);
        const double t = time(split > 1 ? 7.0 : 5.5, r * ((double)((groups + split - 1) / split) * step_us[i] + 0.4));
        if (t < best) { best = t; best_nt = nts[i]; best_split = split; }
    }
    switch (best_nt) {
        case 16: return launch_form<16>(a, best_split, s);
        case 32: return launch_form<32>(a, best_split, s);
        case 64: return launch_form<64>(a, best_split, s);
        default: return launch_block_mm_pair(a, best_split, s);
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
