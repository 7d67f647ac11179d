// Quantisation to e4m3 with a scale for each 128 values of a row (activations) or each 128 x 128 block (weights).
//
// Bound by memory: one read of the source, one byte written per value.  Rows: a warp takes one unit of four adjacent rows at
// a time (a unit is 256 columns in 16-byte accesses for 16-bit data, 128 otherwise), whose scales lie side by side, with the
// next four on their way; a reduction over lanes per 128-column block.  Weights: a CTA takes one block and keeps it in
// registers between the reduction and the output; of fp32 weights each warp has 16 rows, of 16-bit ones half a warp eight.
#pragma once
#include "qssm_elem.cuh"

namespace qssm {

struct QuantParams {
    const void* x;
    uint8_t* q;
    float* scales;
    long long rows, x_stride, q_stride, scale_row, scale_blk;
    int K;
    bool q_words;  // rows of q start on 16-byte boundaries
};

constexpr int QUANT_ROWS = 4;  // rows whose unit a warp takes at a time

// One unit of a row as it lies in memory (16-bit elements two to a register), zeros outside.
template <typename T, int V> struct QuantUnit {
    static constexpr int EPT = V == 8 ? 8 : 4, COLS = 32 * EPT, ACC = EPT / V, BYTES = V * (int)sizeof(T);
    using W = typename Word<BYTES>::type;
    alignas(16) T e[EPT];
    __device__ __forceinline__ void load(const T* row, int unit, int lane, int cols) {
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            const int col = unit * COLS + a * 32 * V + lane * V;
            W w{};
            if (col < cols) w = *reinterpret_cast<const W*>(row + col);
            reinterpret_cast<W*>(e)[a] = w;
        }
    }
    __device__ __forceinline__ void take(QuantUnit& to) { to = *this; }
    // the largest magnitude, NaN if there is one; 16-bit types two at a time
    __device__ __forceinline__ float amax() const {
        if constexpr (std::is_same<T, float>::value) {
            float m = fabsf(e[0]);
#pragma unroll
            for (int i = 1; i < EPT; ++i) m = max_nan(m, fabsf(e[i]));
            return m;
        } else {
            using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            const T2* v = reinterpret_cast<const T2*>(e);
            T2 m = __habs2(v[0]);
#pragma unroll
            for (int i = 1; i < EPT / 2; ++i) m = __hmax2_nan(m, __habs2(v[i]));
            return max_nan(to_f32(m.x), to_f32(m.y));
        }
    }
    __device__ __forceinline__ void store(uint8_t* row, int unit, int lane, int cols, const Fp8Scale& by) const {
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            const int col = unit * COLS + a * 32 * V + lane * V;
            float t[V];
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = to_f32(e[a * V + i]);
            if (col < cols) store_fp8<V>(row + col, t, by);
        }
    }
};

// A unit on its way: as it lies in memory too, but for 16-bit elements that come one or two at a time.
template <typename T, int V> struct SingleQuant : Singles<T, V, QuantUnit<T, V>::EPT> {
    using Base = Singles<T, V, QuantUnit<T, V>::EPT>;
    __device__ __forceinline__ void load(const T* row, int unit, int lane, int cols) {
#pragma unroll
        for (int a = 0; a < QuantUnit<T, V>::ACC; ++a) {
            const int col = unit * QuantUnit<T, V>::COLS + a * 32 * V + lane * V;
            Base::load(a, row + col, col < cols);
        }
    }
    __device__ __forceinline__ void take(QuantUnit<T, V>& to) { Base::take(to.e); }
};
template <typename T, int V>
using QuantComing = typename std::conditional<V <= 2 && sizeof(T) == 2, SingleQuant<T, V <= 2 ? V : 1>, QuantUnit<T, V>>::type;

template <typename T, int V> __global__ void __launch_bounds__(256) quant_rows_kernel(const QuantParams p) {
    using U = QuantUnit<T, V>;
    constexpr int N = QUANT_ROWS, BPU = V == 8 ? 2 : 1, NB = N * BPU;  // blocks of a unit, of a warp's turn
    const int lane = threadIdx.x & 31;
    const int units = (p.K + U::COLS - 1) / U::COLS;
    const long long jobs = (p.rows + N - 1) / N * units, step = (long long)gridDim.x * 8;
    long long job = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (job >= jobs) return;
    U now[N];
    QuantComing<T, V> next[N];
    auto fetch = [&](long long row, int unit) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            next[i].load(static_cast<const T*>(p.x) + (row + i) * p.x_stride, unit, lane, row + i < p.rows ? p.K : 0);
    };
    auto take = [&]() {
#pragma unroll
        for (int i = 0; i < N; ++i) next[i].take(now[i]);
    };
    long long row = job / units * N;
    int unit = (int)(job % units);
    fetch(row, unit);
    take();
    for (;;) {  // the next units are on their way while these are worked on
        job += step;
        const long long row1 = job < jobs ? job / units * N : p.rows;
        const int unit1 = job < jobs ? (int)(job % units) : 0;
        fetch(row1, unit1);
        // every lane learns the blocks' largest magnitudes, one lane for each block turns its own into the scale
        const int mine = lane & (NB - 1), i = mine / BPU, block = unit * BPU + mine % BPU;
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float m = now[k].amax();
#pragma unroll
            for (int b = 0; b < BPU; ++b) {
                const float all = max_lanes<32>(BPU == 1 || (lane >> 4) == b ? m : 0.f);
                if (mine == k * BPU + b) amax = all;
            }
        }
        const float scale = fp8_scale(amax);
        const Fp8Scale by(scale);
#pragma unroll
        for (int k = 0; k < N; ++k)
            now[k].store(p.q + (row + k) * p.q_stride, unit, lane, row + k < p.rows ? p.K : 0,
                         by.from_lane(k * BPU + (BPU == 2 ? lane >> 4 : 0)));
        if (lane < NB && row + i < p.rows && block * FP8_BLOCK < p.K)
            p.scales[(row + i) * p.scale_row + (long long)block * p.scale_blk] = scale;
        if (job >= jobs) return;
        row = row1;
        unit = unit1;
        take();
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
    const Fp8Scale by(scale);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const long long row = row0 + warp + 8 * r;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            const int col = col0 + a * 32 * V + lane * V;
            float t[V];
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = v[r][a * V + i];
            if (row < p.rows && col < p.K) store_fp8<V>(p.q + row * p.q_stride + col, t, by);
        }
    }
    if (threadIdx.x == 0) p.scales[(long long)blockIdx.y * p.scale_row + (long long)blockIdx.x * p.scale_blk] = scale;
}

// Blocks of 16-bit weights: eight elements a lane and access, 16 lanes to a row, kept as they came.  ANY: rows start
// anywhere.  65536x1024 bf16 46 us, 65536x1023 58; four (one) at a time 58 (205).  Bound by latency: a CTA has one block,
// and nothing is on its way while that is reduced and written.
template <typename T, bool ANY> __global__ void __launch_bounds__(256) quant_blocks16_kernel(const QuantParams p) {
    constexpr int PER = 16, TIMES = FP8_BLOCK / PER;  // rows at a time
    using U = QuantUnit<T, 8>;
    __shared__ float red[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = threadIdx.x & 15, col0 = blockIdx.x * FP8_BLOCK;
    const int cols = p.K - col0 < FP8_BLOCK ? p.K - col0 : FP8_BLOCK;
    const long long row0 = (long long)blockIdx.y * FP8_BLOCK + (threadIdx.x >> 4);
    U v[TIMES];
    float amax = 0.f;
    // the source's first and last block do without words that reach over its ends (two loops: a choice in each row's turn
    // keeps the rows' loads from being under way together, 65536x1023 85 us against 60)
    const long long top = (long long)blockIdx.y * FP8_BLOCK, bottom = top + FP8_BLOCK < p.rows ? top + FP8_BLOCK : p.rows;
    const bool words = !ANY || words_inside(top * p.x_stride + col0, (bottom - 1) * p.x_stride + col0 + cols,
                                            (p.rows - 1) * p.x_stride + p.K);
    auto load = [&](auto any) {
#pragma unroll
        for (int r = 0; r < TIMES; ++r) {
            const long long row = row0 + PER * r;
            const T* at = static_cast<const T*>(p.x) + row * p.x_stride + col0;
            const int here = row < p.rows ? cols : 0;
            if constexpr (!ANY) v[r].load(at, 0, l, here);
            else if constexpr (decltype(any)::value) load_any8(at + 8 * l, here - 8 * l, v[r].e);
            else load_each8(at + 8 * l, here - 8 * l, v[r].e);
        }
    };
    if (words) load(std::true_type{});
    else if constexpr (ANY) load(std::false_type{});
#pragma unroll
    for (int r = 0; r < TIMES; ++r) amax = max_nan(amax, v[r].amax());
    amax = max_lanes<32>(amax);
    if (lane == 0) red[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = max_nan(amax, red[k]);
    const float scale = fp8_scale(amax);
    const Fp8Scale by(scale);
#pragma unroll
    for (int r = 0; r < TIMES; ++r) {
        const long long row = row0 + PER * r;
        const int left = (row < p.rows ? cols : 0) - 8 * l;
        uint8_t* q = p.q + row * p.q_stride + col0 + 8 * l;
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = to_f32(v[r].e[i]);
        if constexpr (ANY) store_fp8_part<8>(q, t, by, left, p.q_words);
        else if (left > 0) store_fp8<8>(q, t, by);
    }
    if (threadIdx.x == 0) p.scales[(long long)blockIdx.y * p.scale_row + (long long)blockIdx.x * p.scale_blk] = scale;
}

}  // namespace qssm
