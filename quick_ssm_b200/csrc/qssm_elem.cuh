// Element access for the row kernels (residual norm, block quantisation): groups of 1 to 8 elements of fp32,
// fp16 or bf16 as fp32 values, conversion to e4m3, warp reductions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include <type_traits>

namespace qssm {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two values rounded and packed in one conversion.
template <typename T> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

template <int BYTES> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

// V adjacent elements in one access (two 16-byte ones where they are longer than that).  The address is a multiple
// of the access size.
template <typename T, int V> __device__ __forceinline__ void load_elems(const T* p, float (&v)[V]) {
    constexpr int BYTES = V * (int)sizeof(T);
    if constexpr (BYTES > 16) {
        static_assert(BYTES == 32, "at most two 16-byte accesses");
        float lo[V / 2], hi[V / 2];
        load_elems<T, V / 2>(p, lo);
        load_elems<T, V / 2>(p + V / 2, hi);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) { v[i] = lo[i]; v[V / 2 + i] = hi[i]; }
    } else {
        union { typename Word<BYTES>::type w; T e[V]; } u;
        u.w = *reinterpret_cast<const typename Word<BYTES>::type*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f32(u.e[i]);
    }
}
template <typename T, int V> __device__ __forceinline__ void store_elems(T* p, const float (&v)[V]) {
    constexpr int BYTES = V * (int)sizeof(T);
    if constexpr (BYTES > 16) {
        float lo[V / 2], hi[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) { lo[i] = v[i]; hi[i] = v[V / 2 + i]; }
        store_elems<T, V / 2>(p, lo);
        store_elems<T, V / 2>(p + V / 2, hi);
    } else {
        union U { typename Word<BYTES>::type w; T e[V]; uint32_t p[V > 1 ? V / 2 : 1]; __device__ U() {} } u;
        if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) u.p[i] = pack_pair<T>(v[2 * i], v[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) u.e[i] = from_f32<T>(v[i]);
        }
        *reinterpret_cast<typename Word<BYTES>::type*>(p) = u.w;
    }
}

// N 16-bit elements on their way that come one or two at a time: each access keeps a register of its own until it is
// taken.  Single elements two to a register would have to be joined, and that waits for them where the next rows should
// only be fetched (residual norm of 65536x1023 bf16 258 us against 142, its backward 510 against 260).
template <typename T, int V, int N> struct Singles {
    static_assert(sizeof(T) == 2 && V <= 2, "16-bit elements, one or two");
    using W = typename Word<2 * V>::type;
    uint32_t w[N / V];
    __device__ __forceinline__ void load(int i, const T* p, bool in) {
        w[i] = 0;
        if (in) w[i] = *reinterpret_cast<const W*>(p);
    }
    __device__ __forceinline__ void take(T (&to)[N]) {
#pragma unroll
        for (int i = 0; i < N / V; ++i) {
            asm volatile("" : "+r"(w[i]));
            reinterpret_cast<W*>(to)[i] = (W)w[i];
        }
    }
};

// Eight 16-bit elements from any element's address on, in 16-byte accesses: an aligned word and the one behind it, moved
// into place in registers.  A word that holds one of the `left` elements is read whole: it reaches up to seven elements over
// their ends (`words_inside` says where it may).  Zeros stand for what lies behind them.
template <typename T> __device__ __forceinline__ void load_any8(const T* p, int left, T (&out)[8]) {
    const int s = (int)(reinterpret_cast<uintptr_t>(p) >> 1) & 7;
    const uint4* at = reinterpret_cast<const uint4*>(p - s);
    uint4 lo{}, hi{};
    if (left > 0) lo = at[0];
    if (s > 0 && left > 8 - s) hi = at[1];
    uint32_t a[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) a[i] = s & 4 ? a[i + 2] : a[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) a[i] = s & 2 ? a[i + 1] : a[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = __funnelshift_r(a[i], a[i + 1], (s & 1) * 16);
    if (left < 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = left >= 2 * i + 2 ? a[i] : left == 2 * i + 1 ? a[i] & 0xffffu : 0u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(out)[i] = a[i];
}
// The same one by one.
template <typename T> __device__ __forceinline__ void load_each8(const T* p, int left, T (&out)[8]) {
    const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<uint16_t*>(out)[i] = i < left ? e[i] : (uint16_t)0;
}
// Do the words around the elements from `first` to `last` of a source (counted from its first one) lie between the first and
// the last of its `all` elements, gaps between rows included?
__device__ __forceinline__ bool words_inside(long long first, long long last, long long all) { return first >= 7 && last + 7 <= all; }

__device__ __forceinline__ float sum_warp(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// fmaxf drops a NaN; a block that holds one has to end up NaN as a whole.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The largest of 16 or 32 adjacent lanes' magnitudes.  A whole warp's in one instruction, as bit patterns: magnitudes
// order as unsigned integers, a NaN above infinity.  With a mask for each half that instruction runs twice and is slower
// than shuffles (quantisation of 65536x4096 bf16 193 us against 178).
template <int LANES> __device__ __forceinline__ float max_lanes(float magnitude) {
    if constexpr (LANES == 32) {
        return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(magnitude)));
    } else {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) magnitude = max_nan(magnitude, __shfl_xor_sync(0xffffffffu, magnitude, o));
        return magnitude;
    }
}

// Quantisation of a block: scale = max(amax, 2^-100) / 448 (448 is e4m3's largest value; the floor keeps the scale a
// normal number for blocks of zeros), value = e4m3(v / scale), nearest even.  An infinity in the block makes the scale
// infinite and its own value NaN, a NaN makes the scale NaN: what is computed from such a block is NaN.
constexpr float FP8_MAX = 448.f;
constexpr float FP8_AMAX_FLOOR = 7.888609052210118e-31f;  // 2^-100
constexpr int FP8_BLOCK = 128;

__device__ __forceinline__ unsigned long long& as_u64(float2& v) { return reinterpret_cast<unsigned long long&>(v); }
__device__ __forceinline__ const unsigned long long& as_u64(const float2& v) {
    return reinterpret_cast<const unsigned long long&>(v);
}

// Quotients without divisions (a division for each value bound these kernels at half the copy rate): with r = 1/b rounded,
// q = a r is a unit off at most, and q - (q b - a) r, its residual exact in one fused multiply-add, is the rounded quotient
// (P. Markstein, IBM J. Res. Dev. 34, 1990).
__device__ __forceinline__ float quotient(float a, float b, float r) {
    const float q = a * r;
    return fmaf(-fmaf(q, b, -a), r, q);
}
__device__ __forceinline__ float fp8_scale(float amax) {
    const float m = max_nan(amax, FP8_AMAX_FLOOR), s = quotient(m, FP8_MAX, 1.f / FP8_MAX);
    return m <= 3.402823466e38f ? s : m;  // an infinity and a NaN are their own scale
}
// 1/scale: the hardware's estimate and one Newton step.  An infinite scale makes every finite value zero: its reciprocal
// is zero, and the largest finite number in its place keeps the residuals finite.
struct Fp8Scale {
    float s, r;
    __device__ __forceinline__ explicit Fp8Scale(float scale) {
        s = scale < 3.402823466e38f ? scale : 3.402823466e38f;
        float e;
        asm("rcp.approx.f32 %0, %1;" : "=f"(e) : "f"(s));
        r = fmaf(fmaf(-s, e, 1.f), e, e);
        if (!(scale < 3.402823466e38f)) r = scale == scale ? 0.f : scale;
    }
    __device__ __forceinline__ Fp8Scale(float s_, float r_) : s(s_), r(r_) {}
    __device__ __forceinline__ Fp8Scale from_lane(int lane) const {
        return Fp8Scale(__shfl_sync(0xffffffffu, s, lane), __shfl_sync(0xffffffffu, r, lane));
    }
    // -v / scale: in these signs a zero keeps its own, and two values go through one instruction
    __device__ __forceinline__ float minus_of(float v) const {
        const float q = v * -r;
        return fmaf(fmaf(q, s, v), -r, q);
    }
    __device__ __forceinline__ float2 minus_of(float2 v) const {
        const float2 nr = make_float2(-r, -r), s2 = make_float2(s, s);
        float2 q, e;
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(as_u64(q)) : "l"(as_u64(v)), "l"(as_u64(nr)));
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(as_u64(e)) : "l"(as_u64(q)), "l"(as_u64(s2)), "l"(as_u64(v)));
        asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(as_u64(q)) : "l"(as_u64(e)), "l"(as_u64(nr)));
        return q;
    }
};

// Quantised values; the sign that `minus_of` turns is turned back in the bytes.
template <int V> __device__ __forceinline__ void store_fp8(uint8_t* p, const float (&v)[V], const Fp8Scale& scale) {
    if constexpr (V == 1) {
        *p = __nv_cvt_float_to_fp8(scale.minus_of(v[0]), __NV_SATFINITE, __NV_E4M3) ^ 0x80;
    } else {
        union { typename Word<V>::type w; uint16_t h[V / 2]; uint32_t u[V < 4 ? 1 : V / 4]; } u;
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            u.h[i] = __nv_cvt_float2_to_fp8x2(scale.minus_of(make_float2(v[2 * i], v[2 * i + 1])), __NV_SATFINITE, __NV_E4M3);
        if constexpr (V == 2) u.h[0] ^= 0x8080u;
        else {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) u.u[i] ^= 0x80808080u;
        }
        *reinterpret_cast<typename Word<V>::type*>(p) = u.w;
    }
}
// The first `left` of them; byte by byte where the row ends among them or its bytes are not aligned (`words` is false).
template <int V>
__device__ __forceinline__ void store_fp8_part(uint8_t* p, const float (&v)[V], const Fp8Scale& scale, int left, bool words) {
    if (words && left >= V) {
        store_fp8<V>(p, v, scale);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < left) p[i] = __nv_cvt_float_to_fp8(scale.minus_of(v[i]), __NV_SATFINITE, __NV_E4M3) ^ 0x80;
}

}  // namespace qssm
