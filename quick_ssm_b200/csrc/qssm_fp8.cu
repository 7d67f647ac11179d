// Block quantisation to e4m3 and the block-scaled 8-bit product: C entry points.
#include <string.h>

#include "qssm_fp8mm.cuh"
#include "qssm_host.cuh"
#include "qssm_quant.cuh"

using namespace qssm;

namespace {

template <typename F> int with_type(int dtype, F&& f) {
    switch (dtype) {
        case QSSM_F32: return f(float{});
        case QSSM_F16: return f(__half{});
        case QSSM_BF16: return f(__nv_bfloat16{});
        default: return QSSM_E_DTYPE;
    }
}
bool fits(const void* ptr, long long stride, int bytes, int es) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && (stride * es) % bytes == 0;
}
int quant_check(const void* x, const void* q, const void* scales, long long rows, long long K, long long x_stride,
                long long q_stride, int dtype) {
    if (dtype_size(dtype) == 0) return QSSM_E_DTYPE;
    if (rows < 0 || K < 0 || K >= (1ll << 30)) return QSSM_E_SHAPE;
    if (rows == 0 || K == 0) return 0;
    if (x == nullptr || q == nullptr || scales == nullptr) return QSSM_E_NULL;
    if (x_stride < 0 || q_stride < K) return QSSM_E_STRIDE;
    return 0;
}

}  // namespace

extern "C" {

int qssm_quant_fp8_rows(const void* x, void* q, float* scales, int64_t rows, int64_t K, int64_t x_stride,
                        int64_t q_stride, int64_t scale_stride_row, int64_t scale_stride_blk, int dtype, void* stream) {
    const int rc = quant_check(x, q, scales, rows, K, x_stride, q_stride, dtype);
    if (rc || rows == 0 || K == 0) return rc;
    QuantParams p{x, static_cast<uint8_t*>(q), scales, rows, x_stride, q_stride, scale_stride_row, scale_stride_blk, (int)K};
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        constexpr int V = 16 / sizeof(T), COLS = 32 * V;
        const bool vec = K % V == 0 && fits(x, x_stride, 16, sizeof(T)) && fits(q, q_stride, V, 1);
        const long long cols = vec ? COLS : FP8_BLOCK;
        const long long units = (K + cols - 1) / cols, jobs = rows * ((units + QUANT_UNITS - 1) / QUANT_UNITS);
        const long long need = (jobs + 7) / 8, most = 16ll * sm_count();
        const unsigned grid = (unsigned)(need < most ? need : most);
        if (vec) quant_rows_kernel<T, V><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
        else quant_rows_kernel<T, 1><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
        return (int)cudaGetLastError();
    });
}

int qssm_quant_fp8_blocks(const void* w, void* q, float* scales, int64_t N, int64_t K, int64_t w_stride,
                          int64_t q_stride, int64_t scale_stride_row, int64_t scale_stride_blk, int dtype, void* stream) {
    const int rc = quant_check(w, q, scales, N, K, w_stride, q_stride, dtype);
    if (rc || N == 0 || K == 0) return rc;
    if (N > 128ll * 65535) return QSSM_E_SHAPE;
    QuantParams p{w, static_cast<uint8_t*>(q), scales, N, w_stride, q_stride, scale_stride_row, scale_stride_blk, (int)K};
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const bool vec = K % 4 == 0 && fits(w, w_stride, 4 * sizeof(T), sizeof(T)) && fits(q, q_stride, 4, 1);
        const dim3 grid((unsigned)((K + FP8_BLOCK - 1) / FP8_BLOCK), (unsigned)((N + FP8_BLOCK - 1) / FP8_BLOCK));
        if (vec) quant_blocks_kernel<T, 4><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
        else quant_blocks_kernel<T, 1><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
        return (int)cudaGetLastError();
    });
}

int qssm_matmul_fp8(const void* x, const float* x_scales, const void* w, const float* w_scales, const void* bias,
                    void* y, int64_t M, int64_t N, int64_t K, int64_t x_stride, int64_t xs_stride_row,
                    int64_t xs_stride_blk, int64_t w_stride, int64_t ws_stride_row, int64_t ws_stride_blk,
                    int64_t y_stride, int out_dtype, int bias_dtype, int* status_word, void* stream) {
    if (dtype_size(out_dtype) == 0 || (bias != nullptr && dtype_size(bias_dtype) == 0)) return QSSM_E_DTYPE;
    if (M < 0 || N < 0 || K < 0 || M >= (1ll << 31) - 256 || N >= (1ll << 31) - 256 || K >= (1ll << 30)) return QSSM_E_SHAPE;
    if (M == 0 || N == 0) return 0;
    if (y == nullptr || (K > 0 && (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr)))
        return QSSM_E_NULL;
    if (y_stride < N || (K > 0 && (x_stride < K || w_stride < K || !fits(x, x_stride, 16, 1) || !fits(w, w_stride, 16, 1))))
        return QSSM_E_STRIDE;
    MatmulParams p;
    memset(&p, 0, sizeof(p));
    p.x = static_cast<const uint8_t*>(x); p.w = static_cast<const uint8_t*>(w);
    p.x_scales = x_scales; p.w_scales = w_scales; p.bias = bias; p.y = y;
    p.M = M; p.N = N; p.K = K;
    p.x_stride = x_stride; p.xs_row = xs_stride_row; p.xs_blk = xs_stride_blk;
    p.w_stride = w_stride; p.ws_row = ws_stride_row; p.ws_blk = ws_stride_blk; p.y_stride = y_stride;
    p.bias_dtype = bias_dtype; p.status = status_word;
    return with_type(out_dtype, [&](auto t) -> int {
        using T = decltype(t);
        const dim3 grid((unsigned)((N + 15) / 16), (unsigned)((M + 15) / 16));
        if (grid.y > 65535u) return QSSM_E_SHAPE;
        matmul_fp8_plain_kernel<T><<<grid, dim3(16, 16), 0, static_cast<cudaStream_t>(stream)>>>(p);
        return (int)cudaGetLastError();
    });
}

}  // extern "C"
