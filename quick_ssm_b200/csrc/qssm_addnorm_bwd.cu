// Residual sum and RMS norm, backward: C entry point.
#include <string.h>

#include "qssm_addnorm_host.cuh"

using namespace qssm;

extern "C" {

size_t qssm_add_rmsnorm_workspace_bytes(int64_t rows, int64_t H) {
    if (rows <= 0 || H <= 0) return 0;
    const int64_t most = (int64_t)ADDNORM_CTAS * sm_count();
    return (size_t)(rows < most ? rows : most) * (size_t)H * sizeof(float);
}

int qssm_add_rmsnorm_bwd(const void* h, const void* w, const void* dy, const void* dh, const float* rstd, void* dx,
                         void* dres, void* dw, void* ws, size_t ws_bytes, int64_t rows, int64_t H, int64_t h_stride,
                         int64_t dy_stride, int64_t dh_stride, int64_t dx_stride, int64_t dres_stride, int x_dtype,
                         int res_dtype, int w_dtype, void* stream_v) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const int rc = addnorm_check(rows, H, x_dtype, res_dtype, w_dtype);
    if (rc) return rc;
    if (H == 0) return 0;
    if (dw == nullptr) return QSSM_E_NULL;
    if (rows == 0) return (int)cudaMemsetAsync(dw, 0, (size_t)H * dtype_size(w_dtype), stream);
    if (h == nullptr || w == nullptr || dy == nullptr || rstd == nullptr || ws == nullptr ||
        (dx == nullptr && dres == nullptr))
        return QSSM_E_NULL;
    if (h_stride < 0 || dy_stride < 0 || (dh != nullptr && dh_stride < 0) || (dx != nullptr && dx_stride < H) ||
        (dres != nullptr && dres_stride < H))
        return QSSM_E_STRIDE;
    if (reinterpret_cast<uintptr_t>(ws) % 16 != 0 || ws_bytes < qssm_add_rmsnorm_workspace_bytes(rows, H))
        return QSSM_E_WS;
    AddNormParams p;
    memset(&p, 0, sizeof(p));
    p.h = const_cast<void*>(h); p.w = w; p.dy = dy; p.dh = dh; p.rstd = const_cast<float*>(rstd);
    p.dx = dx; p.dres = dres; p.dw_part = static_cast<float*>(ws);
    p.rows = rows; p.H = (int)H;
    p.h_stride = h_stride; p.dy_stride = dy_stride; p.dh_stride = dh_stride; p.dx_stride = dx_stride;
    p.dres_stride = dres_stride;
    p.w_dtype = w_dtype;
    p.w_vec = w_dtype == QSSM_F32 && reinterpret_cast<uintptr_t>(w) % 16 == 0;
    const int es = dtype_size(x_dtype), rs = dtype_size(res_dtype);
    const int V = addnorm_access(es, rs, H, [&](int v) {
        return addnorm_fits(h, h_stride, rs, v) && addnorm_fits(dy, dy_stride, es, v) && addnorm_fits(dh, dh_stride, rs, v) &&
               addnorm_fits(dx, dx_stride, es, v) && addnorm_fits(dres, dres_stride, rs, v);
    });
    int n_part = 0;
    const int err = addnorm_types(x_dtype, res_dtype, [&](auto tx, auto tr) -> int {
        using TX = decltype(tx);
        using TR = decltype(tr);
        return addnorm_variant<TX, TR>(V, rows, (int)H, [&](auto v, auto wpr, auto nu, auto at_once) -> int {
            constexpr int W = decltype(wpr)::value, NU = decltype(nu)::value, R = decltype(at_once)::value,
                          ROWS = ADDNORM_WARPS / W * R;
            p.dw_held = NU == 0 && H * 4 <= ADDNORM_HELD_DW;
            const int smem = (W < ADDNORM_WARPS && NU > 0) || p.dw_held ? (int)H * 4 : 0;  // at most 16 KB but for long rows
            const int room = 227 * 1024 / (smem + 1024), ctas = room < ADDNORM_CTAS ? room : ADDNORM_CTAS;  // of an SM
            const long long need = (rows + ROWS - 1) / ROWS, most = (long long)ctas * sm_count();
            n_part = (int)(need < most ? need : most);
            auto kernel = addnorm_bwd_kernel<TX, TR, decltype(v)::value, W, NU, R>;
            if (NU == 0) {  // by itself the runtime may leave shared memory for fewer CTAs than fit
                int e = p.dw_held ? ensure_smem(kernel, ADDNORM_HELD_DW) : 0;
                if (e == 0)
                    e = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, p.dw_held ? 100 : -1);
                if (e) return e;
            }
            kernel<<<(unsigned)n_part, 32 * ADDNORM_WARPS, smem, stream>>>(p);
            return (int)cudaGetLastError();
        });
    });
    if (err) return err;
    const unsigned grid = (unsigned)((H + 31) / 32);
    if (w_dtype == QSSM_F32)
        addnorm_dw_kernel<float><<<grid, 1024, 0, stream>>>(p.dw_part, static_cast<float*>(dw), n_part, (int)H);
    else if (w_dtype == QSSM_F16)
        addnorm_dw_kernel<__half><<<grid, 1024, 0, stream>>>(p.dw_part, static_cast<__half*>(dw), n_part, (int)H);
    else
        addnorm_dw_kernel<__nv_bfloat16><<<grid, 1024, 0, stream>>>(p.dw_part, static_cast<__nv_bfloat16*>(dw), n_part, (int)H);
    return (int)cudaGetLastError();
}

}  // extern "C"
