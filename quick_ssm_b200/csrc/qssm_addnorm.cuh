// Residual sum and RMS norm in one pass, forward (16/32-bit or e4m3 output) and backward.
//
//     h = x + residual (rounded to the residual's type)      r = 1 / sqrt(mean(h^2) + eps)      y = h * r * w
//     d = dh + r * (w*dy) - h * r^3 * mean(h * w*dy)         dx = dres = d                      dw = sum over rows of dy * h * r
//
// h is rounded where it is stored, and the norm is taken of the stored values: the backward, and the next block,
// see the h that the norm saw.  Sums, r and the arithmetic in between are fp32.
//
// All of it is bound by memory: forward 2 reads and 2 writes per element, backward 3 reads and one write (two if x
// and the residual differ in type).  A row is owned by 1, 2, 4 or 8 warps of a CTA and stays in registers between its
// sum of squares and its output, so nothing is read twice; rows of more elements than eight warps' registers hold are
// read again from the h that was just written (L1/L2).
//
// Columns are dealt to lanes in units: with V = 8 elements per access (16-bit data) a unit is 256 columns, lane l
// owning columns 8l..8l+7; with V <= 4 it is 128 columns in 4/V accesses of V adjacent elements per lane.  Either way
// a 128-column quantisation block lies in one access group of 16 or 32 lanes, and its largest magnitude is a shuffle
// reduction.  V = 4 serves what has fp32 in it and short rows of 16 bits, V = 2 and 1 rows whose pitch or length allow
// no more.
//
// A lane holds 16 elements of a row (the backward keeps three values of each, packed as they came, and the dw sums), which
// leaves room for 16 to 32 warps on an SM; a warp takes several rows of one unit at a time.
// Measured on a B200 against the copy rate (6.54 TB/s), bf16 65536x1024: forward 89 us of 82, to e4m3 84 of 72,
// backward 104 of 82 (32 elements a lane as floats, eight warps on an SM: 187; the next row not fetched ahead: 113, and
// to e4m3 104); fp32 165 of 164, 133 of 133, 167 of 164; bf16 on an fp32 stream 125 of 123, 115 of 113, 172 of 164.
#pragma once
#include "qssm_elem.cuh"

namespace qssm {

constexpr int ADDNORM_WARPS = 8;      // warps per CTA
constexpr int ADDNORM_HELD = 16;      // elements of a row that a lane holds in registers
constexpr int ADDNORM_CTAS = 4;       // upper bound of CTAs per SM in the backward (sizes its scratch)

constexpr int ADDNORM_HELD_DW = 72 * 1024;  // bytes of dw sums that a CTA holds, three CTAs on an SM

struct AddNormParams {
    const void* x;
    const void* res;     // NULL: h is x
    const void* w;
    void* y;             // forward: y, or the e4m3 values
    void* h;             // forward: written if res != NULL; backward: read
    float* rstd;         // forward: written if not NULL; backward: read
    float* scales;       // fp8 output
    const void* dy;      // backward
    const void* dh;      // backward, may be NULL
    void* dx;            // backward, may be NULL
    void* dres;          // backward, may be NULL
    float* dw_part;      // backward: [CTAs, H]
    long long rows, x_stride, res_stride, y_stride, h_stride, dy_stride, dh_stride, dx_stride, dres_stride;
    long long scale_row, scale_blk;
    int H, w_dtype, w_vec;
    bool dw_held;        // backward, long rows: shared memory holds the CTA's dw sums
    float eps;
};

template <int V> struct Unit {
    static constexpr int EPT = V == 8 ? 8 : 4;    // elements per lane
    static constexpr int COLS = 32 * EPT;
    static constexpr int ACC = EPT / V;           // accesses per lane
    __device__ static __forceinline__ int col(int unit, int acc, int lane) {
        return unit * COLS + acc * 32 * V + lane * V;
    }
};

template <typename T, int V, int EPT>
__device__ __forceinline__ void load_unit(const T* row, int unit, int lane, int H, float (&v)[EPT]) {
#pragma unroll
    for (int a = 0; a < Unit<V>::ACC; ++a) {
        const int col = Unit<V>::col(unit, a, lane);
        float t[V];
        if (col < H) load_elems<T, V>(row + col, t);
#pragma unroll
        for (int i = 0; i < V; ++i) v[a * V + i] = col < H ? t[i] : 0.f;
    }
}
template <typename T, int V, int EPT>
__device__ __forceinline__ void store_unit(T* row, int unit, int lane, int H, const float (&v)[EPT]) {
#pragma unroll
    for (int a = 0; a < Unit<V>::ACC; ++a) {
        const int col = Unit<V>::col(unit, a, lane);
        float t[V];
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = v[a * V + i];
        if (col < H) store_elems<T, V>(row + col, t);
    }
}
// The weight in its own type (0 fp32, 1 fp16, 2 bf16); 16-byte loads for fp32 weights that allow them.
template <int V, int EPT>
__device__ __forceinline__ void load_weight(const AddNormParams& p, int unit, int lane, float (&v)[EPT]) {
#pragma unroll
    for (int a = 0; a < Unit<V>::ACC; ++a) {
        const int col = Unit<V>::col(unit, a, lane);
        if constexpr (V >= 2) {
            if (p.w_vec) {
                float t[V];
                if (col < p.H) load_elems<float, V>(static_cast<const float*>(p.w) + col, t);
#pragma unroll
                for (int i = 0; i < V; ++i) v[a * V + i] = col < p.H ? t[i] : 0.f;
                continue;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float t = 0.f;
            if (col + i < p.H) {
                if (p.w_dtype == 0) t = static_cast<const float*>(p.w)[col + i];
                else if (p.w_dtype == 1) t = to_f32(static_cast<const __half*>(p.w)[col + i]);
                else t = to_f32(static_cast<const __nv_bfloat16*>(p.w)[col + i]);
            }
            v[a * V + i] = t;
        }
    }
}
// The sum over the row of WPR warps, in warp order.  `red` alternates between two sets, so that one barrier per sum is
// enough; rows of fewer warps than the CTA's have barriers of their own.
template <int WPR> __device__ __forceinline__ float sum_row(float v, float (*red)[ADDNORM_WARPS], int& turn) {
    v = sum_warp(v);
    if constexpr (WPR > 1) {
        const int warp = threadIdx.x >> 5, group = warp / WPR;
        if ((threadIdx.x & 31) == 0) red[turn][warp] = v;
        __syncwarp();  // the barrier wants the warp whole again
        if constexpr (WPR == ADDNORM_WARPS) __syncthreads();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * WPR) : "memory");
        v = 0.f;
#pragma unroll
        for (int k = 0; k < WPR; ++k) v += red[turn][group * WPR + k];
        turn ^= 1;
    }
    return v;
}

// One unit of y, 16/32 bits, or quantised: the lanes of a block agree on its largest magnitude.
template <typename TX, int V, bool FP8, int EPT>
__device__ __forceinline__ void put_unit(const AddNormParams& p, long long row, int unit, int lane, const float (&y)[EPT]) {
    if constexpr (!FP8) {
        store_unit<TX, V>(static_cast<TX*>(p.y) + row * p.y_stride, unit, lane, p.H, y);
    } else {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < EPT; ++i) amax = max_nan(amax, fabsf(y[i]));
        amax = max_lanes<V == 8 ? 16 : 32>(amax);
        const float scale = fp8_scale(amax);
        const Fp8Scale by(scale);
        uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.y_stride;
#pragma unroll
        for (int a = 0; a < Unit<V>::ACC; ++a) {
            const int col = Unit<V>::col(unit, a, lane);
            float t[V];
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = y[a * V + i];
            if (col < p.H) store_fp8<V>(q + col, t, by);
        }
        const int first = Unit<V>::col(unit, 0, lane);
        if ((lane & (V == 8 ? 15 : 31)) == 0 && first < p.H)
            p.scales[row * p.scale_row + (long long)(first / FP8_BLOCK) * p.scale_blk] = scale;
    }
}

// All units that a warp holds of a row, quantised.  Every lane learns all blocks' largest magnitudes; one
// lane for each block turns its own into the scale, which saves the others that arithmetic (60 instructions of 29 for
// four units of 128 columns).
template <int V, int WPR, int N, int EPT>
__device__ __forceinline__ void put_units_fp8(const AddNormParams& p, long long row, int wid, int lane, const float (&y)[N][EPT]) {
    constexpr int BPU = V == 8 ? 2 : 1, NB = N * BPU;  // blocks of a unit, of the row's part
    static_assert((NB & (NB - 1)) == 0, "a power of two");
    const int mine = lane & (NB - 1);
    float amax = 0.f;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        float m = fabsf(y[u][0]);
#pragma unroll
        for (int i = 1; i < EPT; ++i) m = max_nan(m, fabsf(y[u][i]));
#pragma unroll
        for (int b = 0; b < BPU; ++b) {
            const float all = max_lanes<32>(BPU == 1 || (lane >> 4) == b ? m : 0.f);
            if (mine == u * BPU + b) amax = all;
        }
    }
    const float scale = fp8_scale(amax);
    const Fp8Scale by(scale);
    uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.y_stride;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const Fp8Scale s = by.from_lane(u * BPU + (BPU == 2 ? lane >> 4 : 0));
#pragma unroll
        for (int a = 0; a < Unit<V>::ACC; ++a) {
            const int col = Unit<V>::col(u * WPR + wid, a, lane);
            float t[V];
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = y[u][a * V + i];
            if (col < p.H) store_fp8<V>(q + col, t, s);
        }
    }
    const int block = ((mine / BPU) * WPR + wid) * BPU + mine % BPU;
    if (lane < NB && block * FP8_BLOCK < p.H) p.scales[row * p.scale_row + (long long)block * p.scale_blk] = scale;
}

// A unit of a row as it lies in memory (16-bit elements two to a register).
template <typename T, int V> struct Packed {
    static constexpr int EPT = Unit<V>::EPT;
    alignas(16) T e[EPT];
    __device__ __forceinline__ void load(const T* row, int unit, int lane, int cols) {
        constexpr int BYTES = V * (int)sizeof(T) > 16 ? 16 : V * (int)sizeof(T), WORDS = EPT * (int)sizeof(T) / BYTES,
                      PER_ACC = WORDS / Unit<V>::ACC;
        using W = typename Word<BYTES>::type;
        W* w = reinterpret_cast<W*>(e);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            const int col = Unit<V>::col(unit, i / PER_ACC, lane) + (i % PER_ACC) * (BYTES / (int)sizeof(T));
            w[i] = W{};
            if (col < cols) w[i] = *reinterpret_cast<const W*>(row + col);
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return to_f32(e[i]); }
    __device__ __forceinline__ void take(Packed& to) { to = *this; }
};
// A unit on its way: as it lies in memory too, but for 16-bit elements that come one or two at a time.
template <typename T, int V> struct SingleUnit : Singles<T, V, Unit<V>::EPT> {
    using Base = Singles<T, V, Unit<V>::EPT>;
    __device__ __forceinline__ void load(const T* row, int unit, int lane, int cols) {
#pragma unroll
        for (int a = 0; a < Unit<V>::ACC; ++a) {
            const int col = Unit<V>::col(unit, a, lane);
            Base::load(a, row + col, col < cols);
        }
    }
    __device__ __forceinline__ void take(Packed<T, V>& to) { Base::take(to.e); }
};
template <typename T, int V>
using Coming = typename std::conditional<V <= 2 && sizeof(T) == 2, SingleUnit<T, V <= 2 ? V : 1>, Packed<T, V>>::type;

// WPR: warps per row.  NU: units of a row held in registers by each of its warps, 0 for rows that are longer.  R: rows at
// a time.
template <typename TX, typename TR, int V, int WPR, int NU, int R, bool FP8>
__global__ void __launch_bounds__(32 * ADDNORM_WARPS) addnorm_fwd_kernel(const AddNormParams p) {
    constexpr int EPT = Unit<V>::EPT, N = NU > 0 ? NU : 1;
    static_assert(R == 1 || WPR == 1, "several rows at a time are a warp's own");
    __shared__ float red[2][ADDNORM_WARPS];
    int turn = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wid = warp % WPR;
    constexpr int ROWS = ADDNORM_WARPS / WPR;  // row groups of a CTA
    const long long step = (long long)gridDim.x * ROWS * R;
    const int H = p.H;
    const float inv_h = 1.f / (float)H;
    float w[N][EPT];
    if constexpr (NU > 0) {
#pragma unroll
        for (int u = 0; u < N; ++u) load_weight<V>(p, u * WPR + wid, lane, w[u]);
    }
    // rows held in registers: the next ones are on their way while these are worked on
    Packed<TX, V> x[R][N];
    Packed<TR, V> res[R][N];
    Coming<TX, V> x_next[R][N];
    Coming<TR, V> res_next[R][N];
    auto fetch = [&](long long row0) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const long long row = row0 + k;
            const int cols = row < p.rows ? H : 0;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                x_next[k][u].load(static_cast<const TX*>(p.x) + row * p.x_stride, u * WPR + wid, lane, cols);
                if (p.res != nullptr)
                    res_next[k][u].load(static_cast<const TR*>(p.res) + row * p.res_stride, u * WPR + wid, lane, cols);
            }
        }
    };
    auto take = [&]() {
#pragma unroll
        for (int k = 0; k < R; ++k)
#pragma unroll
            for (int u = 0; u < N; ++u) {
                x_next[k][u].take(x[k][u]);
                if (p.res != nullptr) res_next[k][u].take(res[k][u]);
            }
    };
    const long long begin = ((long long)blockIdx.x * ROWS + warp / WPR) * R;
    if constexpr (NU > 0) {
        fetch(begin);
        take();
    }
    for (long long row0 = begin; row0 < p.rows; row0 += step) {
        if constexpr (NU > 0) {
            fetch(row0 + step);
            float h[R][N][EPT];
#pragma unroll
            for (int k = 0; k < R; ++k) {
                TR* hr = static_cast<TR*>(p.h) + (row0 + k) * p.h_stride;
                const int cols = row0 + k < p.rows ? H : 0;
#pragma unroll
                for (int u = 0; u < N; ++u) {
#pragma unroll
                    for (int i = 0; i < EPT; ++i) h[k][u][i] = x[k][u][i];
                    if (p.res != nullptr) {
#pragma unroll
                        for (int i = 0; i < EPT; ++i) h[k][u][i] = to_f32(from_f32<TR>(h[k][u][i] + res[k][u][i]));
                        store_unit<TR, V>(hr, u * WPR + wid, lane, cols, h[k][u]);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < R; ++k) {
                float ss = 0.f;
#pragma unroll
                for (int u = 0; u < N; ++u)
#pragma unroll
                    for (int i = 0; i < EPT; ++i) ss = fmaf(h[k][u][i], h[k][u][i], ss);
                ss = sum_row<WPR>(ss, red, turn);
                if (R > 1 && row0 + k >= p.rows) break;
                const float r = 1.f / sqrtf(ss * inv_h + p.eps);
                if (p.rstd != nullptr && lane == 0 && wid == 0) p.rstd[row0 + k] = r;
#pragma unroll
                for (int u = 0; u < N; ++u) {
#pragma unroll
                    for (int i = 0; i < EPT; ++i) h[k][u][i] *= w[u][i] * r;
                    if constexpr (!FP8) put_unit<TX, V, false>(p, row0 + k, u * WPR + wid, lane, h[k][u]);
                }
                if constexpr (FP8) put_units_fp8<V, WPR>(p, row0 + k, wid, lane, h[k]);
            }
            take();
        } else {
            const TX* xr = static_cast<const TX*>(p.x) + row0 * p.x_stride;
            const TR* rr = static_cast<const TR*>(p.res) + row0 * p.res_stride;
            TR* hr = static_cast<TR*>(p.h) + row0 * p.h_stride;
            const int units = (H + Unit<V>::COLS - 1) / Unit<V>::COLS;
            float ss = 0.f;
            for (int u = wid; u < units; u += WPR) {
                float h[EPT];
                load_unit<TX, V>(xr, u, lane, H, h);
                if (p.res != nullptr) {
                    float t[EPT];
                    load_unit<TR, V>(rr, u, lane, H, t);
#pragma unroll
                    for (int i = 0; i < EPT; ++i) h[i] = to_f32(from_f32<TR>(h[i] + t[i]));
                    store_unit<TR, V>(hr, u, lane, H, h);
                }
#pragma unroll
                for (int i = 0; i < EPT; ++i) ss = fmaf(h[i], h[i], ss);
            }
            ss = sum_row<WPR>(ss, red, turn);
            const float r = 1.f / sqrtf(ss * inv_h + p.eps);
            if (p.rstd != nullptr && lane == 0 && wid == 0) p.rstd[row0] = r;
            for (int u = wid; u < units; u += WPR) {  // a lane reads back what it wrote itself
                float h[EPT], wu[EPT];
                if (p.res != nullptr) load_unit<TR, V>(hr, u, lane, H, h);
                else load_unit<TX, V>(xr, u, lane, H, h);
                load_weight<V>(p, u, lane, wu);
#pragma unroll
                for (int i = 0; i < EPT; ++i) h[i] *= wu[i] * r;
                put_unit<TX, V, FP8>(p, row0, u, lane, h);
            }
        }
    }
}

// Backward.  Each warp keeps the dw sums of its columns: in registers over all its rows (NU > 0), added up over the
// CTA's row groups in order at the end; for longer rows (eight warps each) in shared memory, or, where three CTAs on an SM
// have no room for that, in the CTA's part of the scratch (4096x16384 bf16 205 us against 249 in the scratch, with an fp32
// residual 346 against 392; with two CTAs on an SM shared memory is the slower one: 20480 columns 444 against 412).  What a
// row brings stays packed as it came.
template <typename TX, typename TR, int V, int WPR, int NU, int R>
__global__ void __launch_bounds__(32 * ADDNORM_WARPS) addnorm_bwd_kernel(const AddNormParams p) {
    constexpr int EPT = Unit<V>::EPT, N = NU > 0 ? NU : 1;
    __shared__ float red[2][ADDNORM_WARPS];
    extern __shared__ __align__(16) float dw_sum[];  // WPR < 8 or long rows: H floats
    int turn = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wid = warp % WPR;
    constexpr int ROWS = ADDNORM_WARPS / WPR;
    const long long step = (long long)gridDim.x * ROWS * R;
    const int H = p.H;
    const int units = (H + Unit<V>::COLS - 1) / Unit<V>::COLS;
    const float inv_h = 1.f / (float)H;
    float* part = p.dw_part + (long long)blockIdx.x * H;
    float dw[N][EPT];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
        for (int i = 0; i < EPT; ++i) dw[u][i] = 0.f;
    // long rows: the sums lie in shared memory where that holds them, in the scratch otherwise
    float* const sums = NU == 0 && p.dw_held ? dw_sum : part;
    if constexpr (NU == 0) {
        for (int u = wid; u < units; u += WPR) store_unit<float, V>(sums, u, lane, H, dw[0]);
    }
    // 16-bit rows: the next ones are on their way while these are worked on (with fp32 three more rows of registers cost
    // more warps than that brings)
    constexpr bool AHEAD = sizeof(TR) == 2 && NU > 0 && V >= 4;
    struct Held {
        Packed<TR, V> h[R][N], e[R][N];
        Packed<TX, V> g[R][N];
        float r[R];
    };
    struct Fetched {
        Coming<TR, V> h[R][N], e[R][N];
        Coming<TX, V> g[R][N];
        float r[R];
    };
    // (four 16-bit elements at a time: the same fields moved one by one, 139 us against 169 on 65536x1020)
    constexpr bool SINGLES = (V <= 2 && (sizeof(TX) == 2 || sizeof(TR) == 2)) || (V == 4 && sizeof(TX) == 2 && sizeof(TR) == 2);
    using Next = typename std::conditional<SINGLES, Fetched, Held>::type;
    auto fetch = [&](auto& to, long long row0) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const long long row = row0 + k;
            const int cols = row < p.rows ? H : 0, ecols = p.dh != nullptr ? cols : 0;
            to.r[k] = cols > 0 ? p.rstd[row] : 0.f;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                to.h[k][u].load(static_cast<const TR*>(p.h) + row * p.h_stride, u * WPR + wid, lane, cols);
                to.g[k][u].load(static_cast<const TX*>(p.dy) + row * p.dy_stride, u * WPR + wid, lane, cols);
                to.e[k][u].load(static_cast<const TR*>(p.dh) + row * p.dh_stride, u * WPR + wid, lane, ecols);
            }
        }
    };
    auto take = [&](Held& to, Next& from) {
        if constexpr (!SINGLES) to = from;
        else {
#pragma unroll
            for (int k = 0; k < R; ++k) {
                to.r[k] = from.r[k];
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    from.h[k][u].take(to.h[k][u]);
                    from.g[k][u].take(to.g[k][u]);
                    from.e[k][u].take(to.e[k][u]);
                }
            }
        }
    };
    const long long begin = ((long long)blockIdx.x * ROWS + warp / WPR) * R;
    Held now;
    Next next;
    if constexpr (AHEAD && SINGLES) {
        fetch(next, begin);
        take(now, next);
    } else if constexpr (AHEAD) fetch(now, begin);
    for (long long row0 = begin; row0 < p.rows; row0 += step) {
        if constexpr (NU > 0) {
            if constexpr (AHEAD) fetch(next, row0 + step);
            else if constexpr (SINGLES) {
                fetch(next, row0);
                take(now, next);
            } else fetch(now, row0);
            auto& h = now.h;
            auto& e = now.e;
            auto& g = now.g;
            auto& r = now.r;
            float dot[R];
#pragma unroll
            for (int k = 0; k < R; ++k) dot[k] = 0.f;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                float w[EPT];
                load_weight<V>(p, u * WPR + wid, lane, w);
#pragma unroll
                for (int k = 0; k < R; ++k)
#pragma unroll
                    for (int i = 0; i < EPT; ++i) {
                        dw[u][i] = fmaf(g[k][u][i] * r[k], h[k][u][i], dw[u][i]);
                        dot[k] = fmaf(h[k][u][i], g[k][u][i] * w[i], dot[k]);
                    }
            }
#pragma unroll
            for (int k = 0; k < R; ++k) dot[k] = sum_row<WPR>(dot[k], red, turn) * inv_h * r[k] * r[k] * r[k];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                float w[EPT];
                load_weight<V>(p, u * WPR + wid, lane, w);
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    const long long row = row0 + k;
                    const int cols = row < p.rows ? H : 0;
                    float d[EPT];
#pragma unroll
                    for (int i = 0; i < EPT; ++i)
                        d[i] = e[k][u][i] + fmaf(-h[k][u][i], dot[k], r[k] * (g[k][u][i] * w[i]));
                    if (p.dx != nullptr)
                        store_unit<TX, V>(static_cast<TX*>(p.dx) + row * p.dx_stride, u * WPR + wid, lane, cols, d);
                    if (p.dres != nullptr)
                        store_unit<TR, V>(static_cast<TR*>(p.dres) + row * p.dres_stride, u * WPR + wid, lane, cols, d);
                }
            }
            if constexpr (AHEAD) take(now, next);
        } else {
            const TR* hr = static_cast<const TR*>(p.h) + row0 * p.h_stride;
            const TX* gr = static_cast<const TX*>(p.dy) + row0 * p.dy_stride;
            const TR* er = static_cast<const TR*>(p.dh) + row0 * p.dh_stride;
            TX* dxr = static_cast<TX*>(p.dx) + row0 * p.dx_stride;
            TR* drr = static_cast<TR*>(p.dres) + row0 * p.dres_stride;
            const float r = p.rstd[row0];
            float dot = 0.f;
            for (int u = wid; u < units; u += WPR) {
                float h[EPT], g[EPT], w[EPT], s[EPT];
                load_unit<TR, V>(hr, u, lane, H, h);
                load_unit<TX, V>(gr, u, lane, H, g);
                load_weight<V>(p, u, lane, w);
                load_unit<float, V>(sums, u, lane, H, s);
#pragma unroll
                for (int i = 0; i < EPT; ++i) {
                    dot = fmaf(h[i], g[i] * w[i], dot);
                    s[i] = fmaf(g[i] * r, h[i], s[i]);
                }
                store_unit<float, V>(sums, u, lane, H, s);
            }
            dot = sum_row<WPR>(dot, red, turn);
            const float k = dot * inv_h * r * r * r;
            for (int u = wid; u < units; u += WPR) {
                float h[EPT], g[EPT], w[EPT], e[EPT];
                load_unit<TR, V>(hr, u, lane, H, h);
                load_unit<TX, V>(gr, u, lane, H, g);
                load_weight<V>(p, u, lane, w);
#pragma unroll
                for (int i = 0; i < EPT; ++i) e[i] = 0.f;
                if (p.dh != nullptr) load_unit<TR, V>(er, u, lane, H, e);
#pragma unroll
                for (int i = 0; i < EPT; ++i) e[i] += fmaf(-h[i], k, r * (w[i] * g[i]));
                if (p.dx != nullptr) store_unit<TX, V>(dxr, u, lane, H, e);
                if (p.dres != nullptr) store_unit<TR, V>(drr, u, lane, H, e);
            }
        }
    }
    if constexpr (NU == 0) {
        if (p.dw_held) {
            for (int u = wid; u < units; u += WPR) {
                float s[EPT];
                load_unit<float, V>(sums, u, lane, H, s);
                store_unit<float, V>(part, u, lane, H, s);
            }
        }
    }
    if constexpr (NU > 0 && WPR == ADDNORM_WARPS) {
#pragma unroll
        for (int u = 0; u < N; ++u) store_unit<float, V>(part, u * WPR + wid, lane, H, dw[u]);
    } else if constexpr (NU > 0) {
        __syncthreads();
        for (int k = 0; k < ROWS; ++k) {
            if (warp / WPR == k) {
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    float s[EPT];
#pragma unroll
                    for (int i = 0; i < EPT; ++i) s[i] = 0.f;
                    if (k > 0) load_unit<float, V>(dw_sum, u * WPR + wid, lane, H, s);
#pragma unroll
                    for (int i = 0; i < EPT; ++i) s[i] += dw[u][i];
                    store_unit<float, V>(k + 1 < ROWS ? dw_sum : part, u * WPR + wid, lane, H, s);
                }
            }
            __syncthreads();
        }
    }
}

// dw = the CTAs' partial sums, 32 columns a CTA: thread (tx, ty) adds rows ty, ty + 32, ..., four sums at a time, then
// the 32 sums of a column are added in ty order.  The order does not depend on scheduling.
template <typename TW>
__global__ void __launch_bounds__(1024) addnorm_dw_kernel(const float* part, TW* dw, int n_part, int H) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + tx;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (col < H) {
        const float* at = part + col;
        int q = ty;
        for (; q + 96 < n_part; q += 128) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += at[(long long)(q + 32 * i) * H];
        }
        for (; q < n_part; q += 32) s[0] += at[(long long)q * H];
    }
    red[ty][tx] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (ty == 0 && col < H) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += red[k][tx];
        dw[col] = from_f32<TW>(t);
    }
}

}  // namespace qssm
