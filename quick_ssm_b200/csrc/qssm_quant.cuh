// Quantisation to e4m3 with a scale for each 128 values of a row (activations) or each 128 x 128 block (weights).
//
// Bound by memory: one read of the source, one byte written per value.  Rows: a warp takes up to four adjacent units of a
// row (a unit is 256 columns in 16-byte accesses for 16-bit data, 128 otherwise), all loads first, then a shuffle
// reduction per 128-column block.  Weights: a CTA takes one block, each warp 16 of its rows, and keeps it in registers
// between the reduction and the output.
#pragma once
#include "qssm_elem.cuh"

namespace qssm {

struct QuantParams {
    const void* x;
    uint8_t* q;
    float* scales;
    long long rows, x_stride, q_stride, scale_row, scale_blk;
    int K;
};

constexpr int QUANT_UNITS = 4;  // units a warp has in flight

template <typename T, int V> __global__ void __launch_bounds__(256) quant_rows_kernel(const QuantParams p) {
    constexpr int EPT = V == 8 ? 8 : 4, COLS = 32 * EPT, ACC = EPT / V;
    const int lane = threadIdx.x & 31;
    const int units = (p.K + COLS - 1) / COLS, groups = (units + QUANT_UNITS - 1) / QUANT_UNITS;
    const long long jobs = p.rows * groups, step = (long long)gridDim.x * 8;
    for (long long job = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); job < jobs; job += step) {
        const long long row = job / groups;
        const int u0 = (int)(job - row * groups) * QUANT_UNITS;
        const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
        uint8_t* qr = p.q + row * p.q_stride;
        float v[QUANT_UNITS][EPT];
#pragma unroll
        for (int u = 0; u < QUANT_UNITS; ++u)
#pragma unroll
            for (int a = 0; a < ACC; ++a) {
                const int col = (u0 + u) * COLS + a * 32 * V + lane * V;
                float t[V];
                if (col < p.K) load_elems<T, V>(xr + col, t);
#pragma unroll
                for (int i = 0; i < V; ++i) v[u][a * V + i] = col < p.K ? t[i] : 0.f;
            }
#pragma unroll
        for (int u = 0; u < QUANT_UNITS; ++u) {
            if (u0 + u >= units) break;
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < EPT; ++i) amax = max_nan(amax, fabsf(v[u][i]));
            amax = max_lanes<V == 8 ? 16 : 32>(amax);
            const float scale = fp8_scale(amax);
#pragma unroll
            for (int a = 0; a < ACC; ++a) {
                const int col = (u0 + u) * COLS + a * 32 * V + lane * V;
                float t[V];
#pragma unroll
                for (int i = 0; i < V; ++i) t[i] = v[u][a * V + i];
                if (col < p.K) store_fp8<V>(qr + col, t, scale);
            }
            const int first = (u0 + u) * COLS + lane * V;
            if ((lane & (V == 8 ? 15 : 31)) == 0 && first < p.K)
                p.scales[row * p.scale_row + (long long)(first / FP8_BLOCK) * p.scale_blk] = scale;
        }
    }
}

template <typename T, int V> __global__ void __launch_bounds__(256) quant_blocks_kernel(const QuantParams p) {
    constexpr int ACC = 4 / V, ROWS = FP8_BLOCK / 8;  // rows per warp
    __shared__ float red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col0 = blockIdx.x * FP8_BLOCK;
    const long long row0 = (long long)blockIdx.y * FP8_BLOCK;
    float v[ROWS][4];
    float amax = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const long long row = row0 + warp + 8 * r;
        const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            const int col = col0 + a * 32 * V + lane * V;
            float t[V];
            const bool in = row < p.rows && col < p.K;
            if (in) load_elems<T, V>(xr + col, t);
#pragma unroll
            for (int i = 0; i < V; ++i) v[r][a * V + i] = in ? t[i] : 0.f;
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = max_nan(amax, fabsf(v[r][i]));
    amax = max_lanes<32>(amax);
    if (lane == 0) red[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = max_nan(amax, red[k]);
    const float scale = fp8_scale(amax);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const long long row = row0 + warp + 8 * r;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            const int col = col0 + a * 32 * V + lane * V;
            float t[V];
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = v[r][a * V + i];
            if (row < p.rows && col < p.K) store_fp8<V>(p.q + row * p.q_stride + col, t, scale);
        }
    }
    if (threadIdx.x == 0) p.scales[(long long)blockIdx.y * p.scale_row + (long long)blockIdx.x * p.scale_blk] = scale;
}

}  // namespace qssm
