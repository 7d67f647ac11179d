// Product of e4m3 operands with a scale for each block of 128 along k:
//
//     y[m, n] = bias[n] + sum over blocks kb of  sx[m, kb] * sw[n / 128, kb] * sum over k in kb of  x[m, k] * w[n, k]
//
// Inner sums and the sum over blocks are fp32; the result is rounded once.
#pragma once
#include "qssm_elem.cuh"

namespace qssm {

struct MatmulParams {
    const uint8_t* x;       // [M, K] e4m3, rows x_stride bytes apart
    const uint8_t* w;       // [N, K] e4m3
    const float* x_scales;  // [M, K/128]
    const float* w_scales;  // [N/128, K/128]
    const void* bias;       // [N] or NULL
    void* y;                // [M, N]
    long long M, N, K, x_stride, xs_row, xs_blk, w_stride, ws_row, ws_blk, y_stride;
    int bias_dtype;
    int* status;
};

__device__ __forceinline__ float e4m3_to_f32(uint8_t v) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}
__device__ __forceinline__ float load_bias(const MatmulParams& p, long long n) {
    if (p.bias == nullptr) return 0.f;
    if (p.bias_dtype == 0) return static_cast<const float*>(p.bias)[n];
    if (p.bias_dtype == 1) return to_f32(static_cast<const __half*>(p.bias)[n]);
    return to_f32(static_cast<const __nv_bfloat16*>(p.bias)[n]);
}

// One thread per output, operands of a 16 x 16 tile through shared memory.
template <typename T> __global__ void __launch_bounds__(256) matmul_fp8_plain_kernel(const MatmulParams p) {
    __shared__ float xs[16][129], ws[16][129];
    const int tx = threadIdx.x, ty = threadIdx.y;
    const long long m0 = (long long)blockIdx.y * 16, n0 = (long long)blockIdx.x * 16;
    const long long m = m0 + ty, n = n0 + tx;
    float sum = 0.f;
    for (long long k0 = 0; k0 < p.K; k0 += 128) {
        for (int i = ty * 16 + tx; i < 16 * 128; i += 256) {
            const int r = i >> 7, c = i & 127;
            xs[r][c] = m0 + r < p.M && k0 + c < p.K ? e4m3_to_f32(p.x[(m0 + r) * p.x_stride + k0 + c]) : 0.f;
            ws[r][c] = n0 + r < p.N && k0 + c < p.K ? e4m3_to_f32(p.w[(n0 + r) * p.w_stride + k0 + c]) : 0.f;
        }
        __syncthreads();
        float t = 0.f;
        for (int c = 0; c < 128; ++c) t = fmaf(xs[ty][c], ws[tx][c], t);
        if (m < p.M && n < p.N) {
            const long long kb = k0 / 128;
            sum = fmaf(t, p.x_scales[m * p.xs_row + kb * p.xs_blk] * p.w_scales[(n / 128) * p.ws_row + kb * p.ws_blk], sum);
        }
        __syncthreads();
    }
    if (m < p.M && n < p.N) static_cast<T*>(p.y)[m * p.y_stride + n] = from_f32<T>(sum + load_bias(p, n));
}

}  // namespace qssm
