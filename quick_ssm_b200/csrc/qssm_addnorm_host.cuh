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

// Elements per access for rows of H columns: the largest that `fits(V)` every tensor.  Short rows of 16-bit data take
// units of 128 columns (V = 4): with 256 half of the lanes would have nothing.
template <typename F> int addnorm_access(int es, int rs, long long H, F&& fits) {
    for (int V = es == 2 && rs == 2 && H > 128 ? 8 : 4; V > 1; V /= 2)
        if (H % V == 0 && fits(V)) return V;
    return 1;
}

// Calls f(Int<V>, Int<WPR>, Int<NU>, Int<R>): as few warps per row as hold it, ADDNORM_HELD elements a lane (eight warps
// with twice as many, then a second read, behind that); more warps per row where there are fewer rows than warps to fill
// the GPU (16 per SM); several rows per warp at a time where a row is one unit.
template <typename TX, typename TR, typename F> int addnorm_variant(int V, long long rows, int H, F&& f) {
    auto go = [&](auto v) -> int {
        constexpr int VV = decltype(v)::value, FULL = ADDNORM_HELD / Unit<VV>::EPT;
        const int units = (H + Unit<VV>::COLS - 1) / Unit<VV>::COLS;
        const long long want = 16ll * sm_count();  // warps
        if (units <= 1) return f(v, AnInt<1>{}, AnInt<1>{}, AnInt<FULL>{});
        if (units <= FULL && rows >= want) return f(v, AnInt<1>{}, AnInt<FULL>{}, AnInt<1>{});
        if constexpr (VV >= 4) {
            if (units <= 2 * FULL && 2 * rows >= want) return f(v, AnInt<2>{}, AnInt<FULL>{}, AnInt<1>{});
        }
        if (units <= 4 * FULL && (VV < 4 || 4 * rows >= want)) return f(v, AnInt<4>{}, AnInt<FULL>{}, AnInt<1>{});
        if (units <= 8 * FULL) return f(v, AnInt<8>{}, AnInt<FULL>{}, AnInt<1>{});
        if (units <= 16 * FULL) return f(v, AnInt<8>{}, AnInt<2 * FULL>{}, AnInt<1>{});
        return f(v, AnInt<8>{}, AnInt<0>{}, AnInt<1>{});
    };
    if constexpr (sizeof(TX) == 2 && sizeof(TR) == 2) {
        if (V == 8) return go(AnInt<8>{});
    }
    if (V == 4) return go(AnInt<4>{});
    if (V == 2) return go(AnInt<2>{});
    return go(AnInt<1>{});
}

inline int addnorm_check(long long rows, long long H, int x_dtype, int res_dtype, int w_dtype) {
    if (dtype_size(x_dtype) == 0 || dtype_size(res_dtype) == 0 || dtype_size(w_dtype) == 0) return QSSM_E_DTYPE;
    if (res_dtype != x_dtype && res_dtype != QSSM_F32) return QSSM_E_DTYPE;
    if (rows < 0 || H < 0 || H >= (1ll << 30)) return QSSM_E_SHAPE;
    return 0;
}

}  // namespace qssm
