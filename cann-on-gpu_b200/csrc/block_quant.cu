// Block quantiser: fp8 codes with one fp32 scale per 128 columns, and the same behind a SwiGLU.
//
//   scale = max(max|x| / top, 2^-126) over the block (1 for a block of zeros),   q = fp8(x * (1 / scale))
//
// top = 448 (e4m3) or 57344 (e5m2).  The scale stays in the normal range so that 1 / scale is finite; x * (1 / scale) is
// at most top * (1 + 2^-22), which rounds to top.  Two IEEE divisions per block and one product per element, so the
// codes are those of the formula in fp32, bit for bit.
//
// SwiGLU uses the fast exponential and quotient (a few 2^-23 of the value, against a code's 2^-4): with expf and an IEEE division
// per element the kernel was bound by instruction issue (4099 x 14336 bf16: 83 us).
//
// HBM-bound: each value is read once and each code written once.  A half-warp owns a block: 8 values per lane (one
// 16-byte load of a 16-bit type, two of fp32), the maximum by four shuffles, 8 codes per lane in one 8-byte store.
#include "device_utils.cuh"

namespace qmm {
namespace {

template <bool E5M2> __device__ __forceinline__ uint32_t codes2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}
template <bool E5M2> __device__ __forceinline__ float block_scale(float amax) {
    constexpr float top = E5M2 ? 57344.f : 448.f;
    return amax > 0.f ? fmaxf(__fdiv_rn(amax, top), 1.17549435e-38f) : 1.f;
}

// 8 consecutive elements from x[idx]; with VEC they lie inside the row and the address is 16-byte aligned, else `n` of them do.
template <int T, bool VEC> __device__ __forceinline__ void load8(const void *x, int64_t idx, int n, float (&f)[8]) {
    if constexpr (VEC) {
        if (n <= 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = 0.f;
            return;
        }
        if constexpr (T == ET_F32) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>((const float *)x + idx));
            const float4 b = __ldg(reinterpret_cast<const float4 *>((const float *)x + idx) + 1);
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        } else {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>((const uint16_t *)x + idx));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (T == ET_BF16) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
                else { f[2 * i] = __half2float(__ushort_as_half((unsigned short)(w[i] & 0xFFFFu))); f[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(w[i] >> 16))); }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < n ? load_as_float(x, T, idx + i) : 0.f;
    }
}

// Rows of D; block b covers columns 128 c .. of row r with b = r * kb + c.  UNROLL blocks per half-warp are in flight.
template <int T, bool VEC, bool SWIGLU, bool E5M2, int UNROLL>
__global__ void __launch_bounds__(256) block_quant_kernel(const void *x, uint8_t *q, float *scale_out, uint32_t nblocks, uint32_t kb, int64_t D) {
    const uint32_t b0 = blockIdx.x * (16u * UNROLL) + (threadIdx.x >> 4);
    const int c8 = (threadIdx.x & 15) * 8;
    float f[UNROLL][8], g[SWIGLU ? UNROLL : 1][8];
    int64_t at[UNROLL];
    int left[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint32_t b = b0 + 16u * u, r = b / kb;
        const int64_t col = (int64_t)(b - r * kb) * 128 + c8, rest = D - col;
        left[u] = b < nblocks ? (int)(rest > 8 ? 8 : rest) : 0;
        at[u] = (int64_t)r * D + col;
        const int64_t in = SWIGLU ? at[u] + (int64_t)r * D : at[u];
        load8<T, VEC>(x, in, left[u], f[u]);
        if constexpr (SWIGLU) load8<T, VEC>(x, in + D, left[u], g[u]);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (SWIGLU) f[u][i] = __fdividef(f[u][i], 1.f + __expf(-f[u][i])) * g[u][i];
            m = fmaxf(m, fabsf(f[u][i]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float sc = block_scale<E5M2>(m), inv = __frcp_rn(sc);
        const uint32_t b = b0 + 16u * u;
        if (c8 == 0 && b < nblocks) scale_out[b] = sc;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = codes2<E5M2>(f[u][2 * i] * inv, f[u][2 * i + 1] * inv);
        if constexpr (VEC) {
            if (left[u] > 0) *reinterpret_cast<uint2 *>(q + at[u]) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left[u]) q[at[u] + i] = (uint8_t)(w[i >> 1] >> (8 * (i & 1)));
        }
    }
}

// 128 x 128 blocks (weights, once at load time): a CTA per block, a half-warp every 16th row, the values in registers
// between the maximum and the codes.
template <int T, bool VEC, bool E5M2>
__global__ void __launch_bounds__(256) tile_quant_kernel(const void *x, uint8_t *q, float *scale_out, int64_t rows, uint32_t kb, int64_t D) {
    __shared__ float sh[8];
    const int64_t r0 = (int64_t)(blockIdx.x / kb) * 128, col = (int64_t)(blockIdx.x % kb) * 128 + (threadIdx.x & 15) * 8;
    const int64_t rest = D - col;
    float f[8][8], m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + (threadIdx.x >> 4) + 16 * i;
        load8<T, VEC>(x, r * D + col, r < rows ? (int)(rest > 8 ? 8 : rest) : 0, f[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(f[i][j]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, sh[w]);
    const float sc = block_scale<E5M2>(m), inv = __frcp_rn(sc);
    if (threadIdx.x == 0) scale_out[blockIdx.x] = sc;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r >= rows) continue;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t w = codes2<E5M2>(f[i][j] * inv, f[i][j + 1] * inv);
            if (j < rest) q[r * D + col + j] = (uint8_t)w;
            if (j + 1 < rest) q[r * D + col + j + 1] = (uint8_t)(w >> 8);
        }
    }
}

template <int T, bool VEC, bool E5M2>
cudaError_t launch_typed(const void *x, int64_t row_block, bool swiglu, uint8_t *q, float *scale_out, int64_t rows, int64_t D, cudaStream_t s) {
    const uint32_t kb = (uint32_t)((D + 127) / 128);
    if (row_block == 128) {
        const int64_t n = (rows + 127) / 128 * kb;
        if (n > 0x7fffffffLL) return cudaErrorInvalidValue;
        tile_quant_kernel<T, VEC, E5M2><<<(unsigned)n, 256, 0, s>>>(x, q, scale_out, rows, kb, D);
    } else {
        const int64_t n = rows * kb;
        if (n > 0x7fffffffLL) return cudaErrorInvalidValue;
        if (swiglu) block_quant_kernel<T, VEC, true, E5M2, 1><<<(unsigned)((n + 15) / 16), 256, 0, s>>>(x, q, scale_out, (uint32_t)n, kb, D);
        else block_quant_kernel<T, VEC, false, E5M2, 1><<<(unsigned)((n + 15) / 16), 256, 0, s>>>(x, q, scale_out, (uint32_t)n, kb, D);
    }
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_block_quant(const void *x, int x_type, int64_t row_block, bool swiglu, uint8_t *q, int q_type, float *scale_out,
                               int64_t rows, int64_t D, cudaStream_t s) {
    if (rows <= 0 || D <= 0) return cudaSuccess;
    const bool vec = D % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
    const bool e5 = q_type == ET_E5M2;
#define BQ(T) (vec ? (e5 ? launch_typed<T, true, true>(x, row_block, swiglu, q, scale_out, rows, D, s)    \
                         : launch_typed<T, true, false>(x, row_block, swiglu, q, scale_out, rows, D, s))  \
                   : (e5 ? launch_typed<T, false, true>(x, row_block, swiglu, q, scale_out, rows, D, s)   \
                         : launch_typed<T, false, false>(x, row_block, swiglu, q, scale_out, rows, D, s)))
    if (x_type == ET_BF16) return BQ(ET_BF16);
    if (x_type == ET_F16) return BQ(ET_F16);
    return BQ(ET_F32);
#undef BQ
}

}  // namespace qmm
