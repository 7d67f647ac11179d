// Launch planning shared by the residual-norm translation units: which kernel variant a call takes.
#pragma once
#include "qssm_addnorm.cuh"
#include "qssm_host.cuh"

namespace qssm {

template <int N> using AnInt = std::integral_constant<int, N>;

// Can V elements of `es` bytes be accessed at once in every row of this tensor?
inline bool addnorm_fits(const void* ptr, long long stride, int es, int V) {
    const int bytes = V * es > 16 ? 16 : V * es;
    return ptr == nullptr || (reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && (stride * es) % bytes == 0);
}

// Calls f(TX{}, TR{}) for the run-time types; the residual stream is in x's type or in fp32.
template <typename F> int addnorm_types(int x_dtype, int res_dtype, F&& f) {
    if (res_dtype != x_dtype && res_dtype != QSSM_F32) return QSSM_E_DTYPE;
    switch (x_dtype) {
        case QSSM_F32: return f(float{}, float{});
        case QSSM_F16: return res_dtype == QSSM_F16 ? f(__half{}, __half{}) : f(__half{}, float{});
        case QSSM_BF16:
            return res_dtype == QSSM_BF16 ? f(__nv_bfloat16{}, __nv_bfloat16{}) : f(__nv_bfloat16{}, float{});
        default: return QSSM_E_DTYPE;
    }
}

// Calls f(Int<V>, Int<WPR>, Int<NU>).  One warp per row for rows of up to 256 elements, and up to 1024 where there are
// enough rows to fill the GPU with such warps (16 per SM); eight warps per row otherwise.
template <typename TX, typename TR, typename F> int addnorm_variant(int V, long long rows, int H, F&& f) {
    const bool one_warp = H <= 256 || (H <= 32 * ADDNORM_HELD && rows >= 16ll * sm_count());
    auto go = [&](auto v) -> int {
        constexpr int VV = decltype(v)::value;
        constexpr int FULL = ADDNORM_HELD / Unit<VV>::EPT, QUARTER = FULL / 4;
        const int units = (H + Unit<VV>::COLS - 1) / Unit<VV>::COLS;
        const int held = one_warp ? units : (units + ADDNORM_WARPS - 1) / ADDNORM_WARPS;
        if (one_warp) return held <= QUARTER ? f(v, AnInt<1>{}, AnInt<QUARTER>{}) : f(v, AnInt<1>{}, AnInt<FULL>{});
        if (held <= QUARTER) return f(v, AnInt<ADDNORM_WARPS>{}, AnInt<QUARTER>{});
        if (held <= FULL) return f(v, AnInt<ADDNORM_WARPS>{}, AnInt<FULL>{});
        return f(v, AnInt<ADDNORM_WARPS>{}, AnInt<0>{});
    };
    if constexpr (sizeof(TX) == 2 && sizeof(TR) == 2) {
        if (V == 8) return go(AnInt<8>{});
        if (V == 2) return go(AnInt<2>{});
    } else {
        if (V == 4) return go(AnInt<4>{});
    }
    return go(AnInt<1>{});
}

inline int addnorm_check(long long rows, long long H, int x_dtype, int res_dtype, int w_dtype) {
    if (dtype_size(x_dtype) == 0 || dtype_size(res_dtype) == 0 || dtype_size(w_dtype) == 0) return QSSM_E_DTYPE;
    if (res_dtype != x_dtype && res_dtype != QSSM_F32) return QSSM_E_DTYPE;
    if (rows < 0 || H < 0 || H >= (1ll << 30)) return QSSM_E_SHAPE;
    return 0;
}

}  // namespace qssm
