// Residual sum and RMS norm, forward: C entry points with 16/32-bit and with e4m3 output.
#include <string.h>

#include "qssm_addnorm_host.cuh"

using namespace qssm;

namespace {

template <bool FP8> int run_forward(AddNormParams& p, int x_dtype, int res_dtype, cudaStream_t stream) {
    const int es = dtype_size(x_dtype), rs = dtype_size(res_dtype);
    const bool has_res = p.res != nullptr;
    const int V = addnorm_access(es, rs, p.H, [&](int v) {
        return addnorm_fits(p.x, p.x_stride, es, v) && addnorm_fits(p.y, p.y_stride, FP8 ? 1 : es, v) &&
               (!has_res || (addnorm_fits(p.res, p.res_stride, rs, v) && addnorm_fits(p.h, p.h_stride, rs, v)));
    });
    return addnorm_types(x_dtype, res_dtype, [&](auto tx, auto tr) -> int {
        using TX = decltype(tx);
        using TR = decltype(tr);
        return addnorm_variant<TX, TR>(V, p.rows, p.H, [&](auto v, auto wpr, auto nu, auto at_once) -> int {
            constexpr int W = decltype(wpr)::value, R = decltype(at_once)::value, ROWS = ADDNORM_WARPS / W * R;
            const long long need = (p.rows + ROWS - 1) / ROWS, most = 8ll * sm_count();
            addnorm_fwd_kernel<TX, TR, decltype(v)::value, W, decltype(nu)::value, R, FP8>
                <<<(unsigned)(need < most ? need : most), 32 * ADDNORM_WARPS, 0, stream>>>(p);
            return (int)cudaGetLastError();
        });
    });
}

}  // namespace

extern "C" {

int qssm_add_rmsnorm_fwd(const void* x, const void* res, const void* w, void* y, void* h, float* rstd, int64_t rows,
                         int64_t H, int64_t x_stride, int64_t res_stride, int64_t y_stride, int64_t h_stride,
                         float eps, int x_dtype, int res_dtype, int w_dtype, void* stream) {
    const int rc = addnorm_check(rows, H, x_dtype, res_dtype, w_dtype);
    if (rc) return rc;
    if (rows == 0 || H == 0) return 0;
    if (x == nullptr || res == nullptr || w == nullptr || y == nullptr || h == nullptr) return QSSM_E_NULL;
    if (x_stride < 0 || res_stride < 0 || y_stride < H || h_stride < H) return QSSM_E_STRIDE;
    AddNormParams p;
    memset(&p, 0, sizeof(p));
    p.x = x; p.res = res; p.w = w; p.y = y; p.h = h; p.rstd = rstd;
    p.rows = rows; p.H = (int)H; p.eps = eps;
    p.x_stride = x_stride; p.res_stride = res_stride; p.y_stride = y_stride; p.h_stride = h_stride;
    p.w_dtype = w_dtype;
    p.w_vec = w_dtype == QSSM_F32 && reinterpret_cast<uintptr_t>(w) % 16 == 0;
    return run_forward<false>(p, x_dtype, res_dtype, static_cast<cudaStream_t>(stream));
}

int qssm_add_rmsnorm_fp8(const void* x, const void* res, const void* w, void* q, float* scales, void* h, int64_t rows,
                         int64_t H, int64_t x_stride, int64_t res_stride, int64_t q_stride, int64_t h_stride,
                         int64_t scale_stride_row, int64_t scale_stride_blk, float eps, int x_dtype, int res_dtype,
                         int w_dtype, void* stream) {
    const int rc = addnorm_check(rows, H, x_dtype, res_dtype, w_dtype);
    if (rc) return rc;
    if (rows == 0 || H == 0) return 0;
    if (x == nullptr || w == nullptr || q == nullptr || scales == nullptr || (res != nullptr && h == nullptr))
        return QSSM_E_NULL;
    if (x_stride < 0 || q_stride < H || (res != nullptr && (res_stride < 0 || h_stride < H))) return QSSM_E_STRIDE;
    AddNormParams p;
    memset(&p, 0, sizeof(p));
    p.x = x; p.res = res; p.w = w; p.y = q; p.h = h; p.scales = scales;
    p.rows = rows; p.H = (int)H; p.eps = eps;
    p.x_stride = x_stride; p.res_stride = res_stride; p.y_stride = q_stride; p.h_stride = h_stride;
    p.scale_row = scale_stride_row; p.scale_blk = scale_stride_blk;
    p.w_dtype = w_dtype;
    p.w_vec = w_dtype == QSSM_F32 && reinterpret_cast<uintptr_t>(w) % 16 == 0;
    return run_forward<true>(p, x_dtype, res == nullptr ? x_dtype : res_dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
