// Block-scaled fp8 matmul, dense or per expert:
//
//   out[m,n] = sum_b xs[m,b] * ws[b,n/128] * ( sum_{k in block b} x[m,k] * w[k,n] ),   b = blocks of 128 k's
//
// The bounds-checked kernel for what the tcgen05 kernels (block_mm_tc.cu, block_mm_pair.cu) do not take: rows that are not a multiple of
// 16 bytes, or operands off a 16-byte boundary.
#include "device_utils.cuh"

namespace qmm {
namespace {

// Tile `tile` of the row tiles of all experts (TM rows each, no tile crosses an expert), found by one warp: the experts
// are scanned 32 at a time.  Every lane gets the expert, its first row of the tile and the rows there; false when the
// tiles end before `tile`.  Counts below 0 count as 0, rows end at M.
__device__ __forceinline__ bool find_row_tile(const int64_t *counts, int E, int64_t M, int TM, int64_t tile, int &expert, int64_t &row0, int &rows) {
    const int lane = threadIdx.x & 31;
    int64_t row_base = 0, tile_base = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
        int64_t c = e0 + lane < E ? __ldg((const long long *)counts + e0 + lane) : 0;
        c = c < 0 ? 0 : (c > M ? M : c);
        int64_t end = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += v;
        }
        int64_t lo = row_base + end - c, hi = row_base + end;
        lo = lo < M ? lo : M;
        hi = hi < M ? hi : M;
        const int64_t nt = (hi - lo + TM - 1) / TM;
        int64_t tend = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, tend, o);
            if (lane >= o) tend += v;
        }
        const int64_t tlo = tile_base + tend - nt;
        const unsigned hit = __ballot_sync(0xffffffffu, tile >= tlo && tile < tlo + nt);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int64_t r0 = lo + (tile - tlo) * TM, left = hi - r0;
            expert = e0 + src;
            row0 = __shfl_sync(0xffffffffu, r0, src);
            rows = (int)__shfl_sync(0xffffffffu, left < TM ? left : (int64_t)TM, src);
            return true;
        }
        row_base += __shfl_sync(0xffffffffu, end, 31);
        tile_base += __shfl_sync(0xffffffffu, tend, 31);
    }
    return false;
}

// ---- any size and alignment ----------------------------------------------------------------------
// 64 x 64 outputs per CTA of eight warps (16 x 32 each), a block of 128 k's at a time: codes are fetched four bytes or, where
// rows do not start on four bytes, one byte at a time, widened to fp16 (exact for both fp8 types) and multiplied by
// mma.sync with fp32 sums, which are folded into the output's sums with the block's two scales.  The next block's codes are on
// their way meanwhile.  Bound by the fetches and conversions: 512 x 4100 x 14336 415 us (rows on four bytes) and 512 x 4097 x 14336 653 us (single bytes),
// where scalar multiply-adds took 6.5 and 6.1 ms; 1 x 4100 x 14336 60 us (867).
constexpr int ST = 64, SK = 128, X_PITCH = SK + 8, W_PITCH = ST + 8;   // pitches in halves: rows 16 bytes apart in the banks

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr, bool trans) {
    if (trans) asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four codes p[0 ..], of which `n` exist, the others 0.  WORDS: rows are whole words and start on one.
template <bool WORDS> __device__ __forceinline__ uint32_t codes4(const uint8_t *p, int n) {
    uint32_t v = 0u;
    if constexpr (WORDS) {
        if (n > 0) v = __ldg(reinterpret_cast<const uint32_t *>(p));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) v |= (uint32_t)__ldg(p + i) << (8 * i);
    }
    return v;
}
// As fp16: e5m2 is its upper byte.
__device__ __forceinline__ uint2 widen4(uint32_t v, bool e5m2) {
    if (e5m2) return make_uint2(__byte_perm(v, 0u, 0x1404), __byte_perm(v, 0u, 0x3424));
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v >> 16), __NV_E4M3);
    return make_uint2((uint32_t)a.x | ((uint32_t)a.y << 16), (uint32_t)b.x | ((uint32_t)b.y << 16));
}
template <int T> __device__ __forceinline__ void store_one(void *out, int64_t at, float v) {
    if constexpr (T == ET_F32) ((float *)out)[at] = v;
    else if constexpr (T == ET_F16) ((__half *)out)[at] = __float2half_rn(v);
    else ((__nv_bfloat16 *)out)[at] = __float2bfloat16_rn(v);
}

template <int T, bool NK, bool WORDS>
__global__ void __launch_bounds__(256, 2) block_mm_simple_kernel(const BlockMmArgs p, int64_t m_tiles, int64_t n_tiles) {
    __shared__ __align__(16) uint16_t sx[ST * X_PITCH];
    __shared__ __align__(16) uint16_t sw[SK * W_PITCH > ST * X_PITCH ? SK * W_PITCH : ST * X_PITCH];   // [n][k] or [k][n]
    __shared__ int s_expert, s_rows;
    __shared__ int64_t s_row0;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int wr = (warp & 3) * 16, wc = (warp >> 2) * 32;   // this warp's outputs
    const int64_t kb = (p.K + 127) / 128, nb = (p.N + 127) / 128;
    const bool x5 = p.x_type == ET_E5M2, w5 = p.w_type == ET_E5M2;
    const uint32_t ax = (uint32_t)__cvta_generic_to_shared(sx) + (uint32_t)((wr + (lane & 15)) * X_PITCH + (lane >> 4) * 8) * 2u;
    // 16 columns x 16 k's of the weights per load: [n][k] as stored, [k][n] transposed on the way
    const uint32_t aw = (uint32_t)__cvta_generic_to_shared(sw) +
                        (NK ? (uint32_t)((wc + (lane & 7) + (lane >> 4) * 8) * X_PITCH + ((lane >> 3) & 1) * 8) : (uint32_t)((lane & 15) * W_PITCH + wc + (lane >> 4) * 8)) * 2u;
    for (int64_t tile = blockIdx.x; tile < m_tiles * n_tiles; tile += gridDim.x) {
        const int64_t mt = tile / n_tiles, n0 = (tile - mt * n_tiles) * ST;
        if (p.experts > 0) {
            if (tid < 32) {
                int e = 0, r = 0;
                int64_t r0 = 0;
                const bool ok = find_row_tile(p.group_rows, (int)p.experts, p.M, ST, mt, e, r0, r);
                if (tid == 0) { s_expert = e; s_row0 = r0; s_rows = ok ? r : 0; }
            }
            __syncthreads();
        }
        const int64_t e = p.experts > 0 ? s_expert : 0, m0 = p.experts > 0 ? s_row0 : mt * ST;
        const int rows = p.experts > 0 ? s_rows : (int)(p.M - m0 < ST ? p.M - m0 : ST);
        if (rows > 0) {
            const uint8_t *w = p.w + e * p.K * p.N;
            const float *ws = p.ws + e * kb * nb + (NK ? n0 / 128 * kb : n0 / 128);
            uint32_t rx[8], rw[8];
            // 8 x 256 groups of four codes of each operand: of x and of [n][k] weights every eighth row, of [k][n] every sixteenth
            const int xr = tid >> 5, xc = (tid & 31) * 4, wk = tid >> 4, wn = (tid & 15) * 4;
            const uint8_t *px = p.x + (m0 + xr) * p.K + xc, *pw = NK ? w + (n0 + xr) * p.K + xc : w + wk * p.N + n0 + wn;
            const int n_left = (int)(p.N - n0 < ST ? p.N - n0 : ST);
            auto fetch = [&](int64_t k0) {
                const int k_left = (int)(p.K - k0 < SK ? p.K - k0 : SK);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    rx[i] = codes4<WORDS>(px + k0 + 8 * i * p.K, xr + 8 * i < rows ? k_left - xc : 0);
                    rw[i] = NK ? codes4<WORDS>(pw + k0 + 8 * i * p.K, xr + 8 * i < n_left ? k_left - xc : 0)
                               : codes4<WORDS>(pw + (k0 + 16 * i) * p.N, wk + 16 * i < k_left ? n_left - wn : 0);
                }
            };
            float acc[4][4] = {};
            const int64_t ra = m0 + wr + (lane >> 2), rb = ra + 8;   // this lane's two rows
            const bool a_in = ra - m0 < rows, b_in = rb - m0 < rows;
            fetch(0);
            for (int64_t blk = 0; blk < kb; ++blk) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    *reinterpret_cast<uint2 *>(sx + (xr + 8 * i) * X_PITCH + xc) = widen4(rx[i], x5);
                    *reinterpret_cast<uint2 *>(NK ? sw + (xr + 8 * i) * X_PITCH + xc : sw + (wk + 16 * i) * W_PITCH + wn) = widen4(rw[i], w5);
                }
                __syncthreads();
                if (blk + 1 < kb) fetch((blk + 1) * SK);
                const float sc = __ldg(ws + (NK ? blk : blk * nb));
                const float fa = a_in ? __ldg(p.xs + ra * kb + blk) * sc : 0.f, fb = b_in ? __ldg(p.xs + rb * kb + blk) * sc : 0.f;
                float part[4][4] = {};
#pragma unroll
                for (int ks = 0; ks < SK / 16; ++ks) {
                    uint32_t a[4];
                    ldsm4(a, ax + ks * 32, false);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {         // 16 columns each
                        uint32_t b[4];
                        ldsm4(b, NK ? aw + (uint32_t)(h * 16 * X_PITCH) * 2u + ks * 32 : aw + (uint32_t)(ks * 16 * W_PITCH + h * 16) * 2u, !NK);
                        mma_f16(part[2 * h], a, b[0], b[1]);
                        mma_f16(part[2 * h + 1], a, b[2], b[3]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[j][0] = fmaf(part[j][0], fa, acc[j][0]);
                    acc[j][1] = fmaf(part[j][1], fa, acc[j][1]);
                    acc[j][2] = fmaf(part[j][2], fb, acc[j][2]);
                    acc[j][3] = fmaf(part[j][3], fb, acc[j][3]);
                }
                __syncthreads();                          // the tiles are rewritten for the next block
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t n = n0 + wc + 8 * j + (lane & 3) * 2;
                if (a_in && n < p.N) store_one<T>(p.out, ra * p.N + n, acc[j][0]);
                if (a_in && n + 1 < p.N) store_one<T>(p.out, ra * p.N + n + 1, acc[j][1]);
                if (b_in && n < p.N) store_one<T>(p.out, rb * p.N + n, acc[j][2]);
                if (b_in && n + 1 < p.N) store_one<T>(p.out, rb * p.N + n + 1, acc[j][3]);
            }
        }
        __syncthreads();   // s_* are rewritten for the next tile
    }
}

cudaError_t launch_simple(const BlockMmArgs &p, cudaStream_t s) {
    const int64_t m_tiles = (p.M + ST - 1) / ST + p.experts, n_tiles = (p.N + ST - 1) / ST, all = m_tiles * n_tiles;
    const unsigned g = (unsigned)(all < (1 << 20) ? all : (1 << 20));
    const bool words = p.K % 4 == 0 && (p.w_nk || p.N % 4 == 0) && ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w)) & 3) == 0;
#define BS(T, NK, W) block_mm_simple_kernel<T, NK, W><<<g, 256, 0, s>>>(p, m_tiles, n_tiles)
#define BST(T) (p.w_nk ? (words ? BS(T, true, true) : BS(T, true, false)) : (words ? BS(T, false, true) : BS(T, false, false)))
    if (p.out_type == ET_BF16) BST(ET_BF16);
    else if (p.out_type == ET_F16) BST(ET_F16);
    else BST(ET_F32);
#undef BST
#undef BS
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_block_mm(const BlockMmArgs &p, cudaStream_t s) {
    return block_mm_tc_supported(p) ? launch_block_mm_tc(p, s) : launch_simple(p, s);
}

}  // namespace qmm
