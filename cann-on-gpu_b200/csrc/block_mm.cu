// Block-scaled fp8 matmul, dense or per expert:
//
//   out[m,n] = sum_b xs[m,b] * ws[b,n/128] * ( sum_{k in block b} x[m,k] * w[k,n] ),   b = blocks of 128 k's
//
// The bounds-checked kernel for what the tensor-core kernel (block_mm_tc.cu) does not take: rows that are not a multiple of
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
// 64 x 64 outputs per CTA of 256 threads, 4 x 4 per thread, K in steps of 16 through shared memory; the sum of a block of
// 128 k's is folded into the output's sum with its two scales when the block ends.
constexpr int ST = 64, SK = 16;
__global__ void __launch_bounds__(256) block_mm_simple_kernel(const BlockMmArgs p, int64_t m_tiles, int64_t n_tiles) {
    __shared__ float sa[SK][ST + 1], sb[SK][ST + 1];
    __shared__ int s_expert, s_rows;
    __shared__ int64_t s_row0;
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int64_t kb = (p.K + 127) / 128, nb = (p.N + 127) / 128;
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
            const float *ws = p.ws + e * kb * nb;
            float acc[4][4] = {}, part[4][4] = {};
            for (int64_t k0 = 0; k0 < p.K; k0 += SK) {
                for (int i = tid; i < ST * SK; i += 256) {
                    const int kk = i % SK, mm = i / SK;
                    const int64_t k = k0 + kk;
                    sa[kk][mm] = mm < rows && k < p.K ? load_as_float(p.x, p.x_type, (m0 + mm) * p.K + k) : 0.f;
                    const int nn = p.w_nk ? mm : i % ST, kw = p.w_nk ? kk : i / ST;
                    const int64_t n = n0 + nn, k2 = k0 + kw;
                    sb[kw][nn] = n < p.N && k2 < p.K ? load_as_float(w, p.w_type, p.w_nk ? n * p.K + k2 : k2 * p.N + n) : 0.f;
                }
                __syncthreads();
#pragma unroll
                for (int kk = 0; kk < SK; ++kk) {
                    float a[4], b[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) { a[i] = sa[kk][ty * 4 + i]; b[i] = sb[kk][tx + 16 * i]; }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) part[i][j] += a[i] * b[j];
                }
                __syncthreads();
                if ((k0 + SK) % 128 == 0 || k0 + SK >= p.K) {
                    const int64_t blk = k0 / 128;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float xs = ty * 4 + i < rows ? __ldg(p.xs + (m0 + ty * 4 + i) * kb + blk) : 0.f;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int64_t n = n0 + tx + 16 * j;
                            const float sc = n < p.N ? __ldg(ws + (p.w_nk ? (n / 128) * kb + blk : blk * nb + n / 128)) : 0.f;
                            acc[i][j] += xs * sc * part[i][j];
                            part[i][j] = 0.f;
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t n = n0 + tx + 16 * j;
                    if (ty * 4 + i < rows && n < p.N) store_from_float(p.out, p.out_type, (m0 + ty * 4 + i) * p.N + n, acc[i][j]);
                }
        }
        __syncthreads();   // s_* are rewritten for the next tile
    }
}

cudaError_t launch_simple(const BlockMmArgs &p, cudaStream_t s) {
    const int64_t m_tiles = (p.M + ST - 1) / ST + p.experts, n_tiles = (p.N + ST - 1) / ST, all = m_tiles * n_tiles;
    block_mm_simple_kernel<<<(unsigned)(all < (1 << 20) ? all : (1 << 20)), 256, 0, s>>>(p, m_tiles, n_tiles);
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_block_mm(const BlockMmArgs &p, cudaStream_t s) {
    return block_mm_tc_supported(p) ? launch_block_mm_tc(p, s) : launch_simple(p, s);
}

}  // namespace qmm
