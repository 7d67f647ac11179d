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

// [rows, cols] as the product's copies see it: boxes of 128 bytes x `box_rows` rows in the 128-byte swizzle, zeros
// outside.  Each host thread keeps the maps it encoded last, as the scan does.  dtype: QSSM_* or -1 for bytes.
int matrix_map(CUtensorMap& map, const void* ptr, long long rows, long long cols, long long pitch_bytes, int dtype, int box_rows) {
    struct Key {
        const void* ptr;
        long long rows, cols, pitch;
        int dtype, box;
        bool operator==(const Key& o) const {
            return ptr == o.ptr && rows == o.rows && cols == o.cols && pitch == o.pitch && dtype == o.dtype && box == o.box;
        }
    };
    struct Entry { Key key; CUtensorMap map; };
    static thread_local Entry cache[64];
    static thread_local bool have_context = false;
    const Key key{ptr, rows, cols, pitch_bytes, dtype, box_rows};
    const unsigned long long hash =
        ((unsigned long long)reinterpret_cast<uintptr_t>(ptr) + 64ull * box_rows + rows + dtype) * 0x9E3779B97F4A7C15ull;
    Entry& e = cache[hash >> 58];
    if (e.key == key) {
        map = e.map;
        return 0;
    }
    if (!have_context) {
        ensure_context();
        have_context = true;
    }
    EncodeTiledFn enc = encode_fn();
    if (enc == nullptr) return QSSM_E_DRIVER;
    const CUtensorMapDataType type = dtype == QSSM_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : dtype == QSSM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : dtype == QSSM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const int es = dtype < 0 ? 1 : dtype_size(dtype);
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch_bytes};
    cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows}, estr[2] = {1u, 1u};
    if (enc(&e.map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
        e.key.ptr = nullptr;
        return QSSM_E_STRIDE;
    }
    e.key = key;
    map = e.map;
    return 0;
}

struct MatmulPlan {
    int T;  // rows per tile of the few-rows kernel; 0: the many-rows kernel
    int S;  // CTAs that share a tile's k
    int x_box, w_box;
};

// Which kernel, and over how many CTAs a tile's k is cut: the shortest of these estimates in microseconds, fitted on a
// B200 with CUDA graphs of 20 calls (N x K 1024x4096, 20480x1024, 4096x4096, 300x16384, 16384x512, 2500x1100, M 1 to
// 4096) to an earlier form of the kernels.  Measured since, many-rows / few-rows kernel: 1x20480x1024 14.4 / 7.1,
// 64x1024x4096 18.9 / 7.6, 64x20480x1024 14.6 / 10.6, 128x20480x1024 15.2 / 17.9, 1024x4096x4096 20.9 / 41.2, 512x300x16384
// 58.2 / 15.3, 1537x2500x1100 11.2 / 19.8: the faster one is chosen each time.  The estimates are 6 to 22 % short of the
// many-rows kernel's times (16384x20480x1024 329 of 373) and within 15 % of the few-rows kernel's.
//   many rows: 0.47 per block of k and round of tiles over the pairs of SMs, 0.9 to end a round (0.7, 1.9, 5.6 more where
//              the rows of y take words of 8, 4, 2 bytes only), 3 to begin;
//   few rows:  0.35 to 0.65 per block of k, 1 per round, 4 to begin, 0.6 to join k.  Clusters of 2, 4 and 8 CTAs are
//              resident on about 148, 136 and 112 SMs (a cluster has to fit into one group of SMs).
MatmulPlan plan_matmul(long long M, long long N, int n_kb, double ragged_us) {
    const long long sms = sm_count(), pairs = sms / 2;
    const long long big = ((M + MMR_M - 1) / MMR_M) * ((N + MMR_N - 1) / MMR_N);
    double best = 3.0 + (double)((big + pairs - 1) / pairs) * (0.47 * n_kb + 0.9 + ragged_us);
    MatmulPlan plan{0, 1, 128, 64};
    const int T = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const double per_block = T == 16 ? 0.35 : T == 32 ? 0.4 : T == 64 ? 0.5 : 0.65;
    const long long tiles = ((N + 127) / 128) * ((M + T - 1) / T);
    if ((M + T - 1) / T > 65535) return plan;  // more tiles of rows than a grid has in its second direction
    for (int S = 1; S <= 8 && S <= n_kb; S *= 2) {
        const long long seats = (T <= 64 ? 2 : 1) * (S == 8 ? sms * 3 / 4 : S == 4 ? sms * 11 / 12 : sms);
        const double cost = 4.0 + (double)((tiles * S + seats - 1) / seats) * (per_block * ((n_kb + S - 1) / S) + 1.0) +
                            (S > 1 ? 0.6 : 0.0);
        if (cost < best) {
            best = cost;
            plan = MatmulPlan{T, S, T, 128};
        }
    }
    return plan;
}

template <typename OUT, int T> int launch_few(const MatmulParams& p, int S, cudaStream_t stream) {
    auto kernel = matmul_fp8_few_kernel<OUT, T>;
    const int rc = ensure_smem(kernel, Few<T>::SMEM);
    if (rc) return rc;
    const long long gx = (long long)((p.N + 127) / 128) * S, gy = (p.M + T - 1) / T;
    if (gx >= (1ll << 31)) return QSSM_E_SHAPE;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)gx, (unsigned)gy);
    cfg.blockDim = dim3(Few<T>::THREADS);
    cfg.dynamicSmemBytes = Few<T>::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)S;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, p, S);
}

}  // namespace

extern "C" {

int qssm_quant_fp8_rows(const void* x, void* q, float* scales, int64_t rows, int64_t K, int64_t x_stride,
                        int64_t q_stride, int64_t scale_stride_row, int64_t scale_stride_blk, int dtype, void* stream) {
    const int rc = quant_check(x, q, scales, rows, K, x_stride, q_stride, dtype);
    if (rc || rows == 0 || K == 0) return rc;
    QuantParams p{x, static_cast<uint8_t*>(q), scales, rows, x_stride, q_stride, scale_stride_row, scale_stride_blk, (int)K, fits(q, q_stride, 16, 1)};
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        constexpr int VEC = 16 / sizeof(T);
        int V = K > 128 ? VEC : 4;  // as many elements per access as every row allows; short rows in units of 128
        while (V > 1 && !(K % V == 0 && fits(x, x_stride, V * (int)sizeof(T), sizeof(T)) && fits(q, q_stride, V, 1))) V /= 2;
        const long long cols = V == 8 ? 256 : 128, jobs = (rows + QUANT_ROWS - 1) / QUANT_ROWS * ((K + cols - 1) / cols);
        const long long need = (jobs + 7) / 8, most = 16ll * sm_count();
        const unsigned grid = (unsigned)(need < most ? need : most);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (V == VEC) quant_rows_kernel<T, VEC><<<grid, 256, 0, s>>>(p);
        else if (V == 4) quant_rows_kernel<T, 4><<<grid, 256, 0, s>>>(p);
        else if (V == 2) quant_rows_kernel<T, 2><<<grid, 256, 0, s>>>(p);
        else quant_rows_kernel<T, 1><<<grid, 256, 0, s>>>(p);
        return (int)cudaGetLastError();
    });
}

int qssm_quant_fp8_blocks(const void* w, void* q, float* scales, int64_t N, int64_t K, int64_t w_stride,
                          int64_t q_stride, int64_t scale_stride_row, int64_t scale_stride_blk, int dtype, void* stream) {
    const int rc = quant_check(w, q, scales, N, K, w_stride, q_stride, dtype);
    if (rc || N == 0 || K == 0) return rc;
    if (N > 128ll * 65535) return QSSM_E_SHAPE;
    QuantParams p{w, static_cast<uint8_t*>(q), scales, N, w_stride, q_stride, scale_stride_row, scale_stride_blk, (int)K, fits(q, q_stride, 16, 1)};
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const dim3 grid((unsigned)((K + FP8_BLOCK - 1) / FP8_BLOCK), (unsigned)((N + FP8_BLOCK - 1) / FP8_BLOCK));
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        constexpr int VEC = 16 / sizeof(T);
        const bool vec = K % VEC == 0 && fits(w, w_stride, 16, sizeof(T)) && fits(q, q_stride, VEC, 1);
        if constexpr (VEC == 8) {
            if (vec) quant_blocks16_kernel<T, false><<<grid, 256, 0, s>>>(p);
            else quant_blocks16_kernel<T, true><<<grid, 256, 0, s>>>(p);
        } else {
            if (vec) quant_blocks_kernel<T, 4><<<grid, 256, 0, s>>>(p);
            else quant_blocks_kernel<T, 1><<<grid, 256, 0, s>>>(p);
        }
        return (int)cudaGetLastError();
    });
}

int qssm_matmul_fp8(const void* x, const float* x_scales, const void* w, const float* w_scales, const void* bias,
                    void* y, int64_t M, int64_t N, int64_t K, int64_t x_stride, int64_t xs_stride_row,
                    int64_t xs_stride_blk, int64_t w_stride, int64_t ws_stride_row, int64_t ws_stride_blk,
                    int64_t y_stride, int out_dtype, int bias_dtype, int* status_word, void* stream_v) {
    if (dtype_size(out_dtype) == 0 || (bias != nullptr && dtype_size(bias_dtype) == 0)) return QSSM_E_DTYPE;
    if (M < 0 || N < 0 || K < 0 || M >= (1ll << 31) - 256 || N >= (1ll << 31) - 256 || K >= (1ll << 30)) return QSSM_E_SHAPE;
    if (M == 0 || N == 0) return 0;
    if (K == 0) return QSSM_E_SHAPE;
    if (y == nullptr || x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr) return QSSM_E_NULL;
    if (y_stride < N || x_stride < K || w_stride < K || !fits(x, x_stride, 16, 1) || !fits(w, w_stride, 16, 1))
        return QSSM_E_STRIDE;
    MatmulParams p;
    memset(&p, 0, sizeof(p));
    p.x_scales = x_scales; p.w_scales = w_scales; p.bias = bias; p.y = y;
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.n_kb = (int)((K + MM_TILE_K - 1) / MM_TILE_K);
    p.xs_row = xs_stride_row; p.xs_blk = xs_stride_blk; p.ws_row = ws_stride_row; p.ws_blk = ws_stride_blk;
    p.y_stride = y_stride;
    p.bias_dtype = bias_dtype; p.status = status_word;
    const int es = dtype_size(out_dtype);
    p.y_vec = fits(y, y_stride, 16, es);
    p.y_word = fits(y, y_stride, 8, es) && N * es % 8 == 0 ? 8 : fits(y, y_stride, 4, es) && N * es % 4 == 0 ? 4 : 2;
    const MatmulPlan plan = plan_matmul(M, N, p.n_kb, p.y_vec ? 0.0 : p.y_word == 8 ? 0.7 : p.y_word == 4 ? 1.9 : 5.6);
    int rc;
    if ((rc = matrix_map(p.x_map, x, M, K, x_stride, -1, plan.x_box)) ||
        (rc = matrix_map(p.w_map, w, N, K, w_stride, -1, plan.w_box)))
        return rc;
    if (plan.T == 0 && p.y_vec && (rc = matrix_map(p.y_map, y, M, N, y_stride * es, out_dtype, 32))) return rc;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    return with_type(out_dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (plan.T == 0) {
            p.m_tiles = (int)((M + MMR_M - 1) / MMR_M);
            p.n_tiles = (int)((N + MMR_N - 1) / MMR_N);
            const long long tiles = (long long)p.m_tiles * p.n_tiles;
            if (tiles >= (1ll << 31) - 1024) return QSSM_E_SHAPE;
            if ((rc = ensure_smem(matmul_fp8_rows_kernel<T>, MMR_SMEM))) return rc;
            const int pairs = sm_count() / 2;
            const unsigned grid = 2u * (unsigned)(tiles < pairs ? tiles : pairs);
            matmul_fp8_rows_kernel<T><<<grid, MMR_THREADS, MMR_SMEM, stream>>>(p);
            return (int)cudaGetLastError();
        }
        switch (plan.T) {
            case 16: return launch_few<T, 16>(p, plan.S, stream);
            case 32: return launch_few<T, 32>(p, plan.S, stream);
            case 64: return launch_few<T, 64>(p, plan.S, stream);
            default: return launch_few<T, 128>(p, plan.S, stream);
        }
    });
}

}  // extern "C"
