// Product of e4m3 operands with a scale for each block of 128 along k:
//
//     y[m, n] = bias[n] + sum over blocks kb of  sx[m, kb] * sw[n / 128, kb] * sum over k in kb of  x[m, k] * w[n, k]
//
// The inner sum of a block is four tcgen05 products of 32 along k into tensor memory; the scales are not powers of
// two in general, so each block's result is read back (tcgen05.ld) and added to fp32 sums in registers with its scale
// while the tensor cores work on the next block in the other buffer.  Inner sums and the sum over blocks are fp32;
// the result is rounded once.
//
// Roles: a warp issues the bulk copies (TMA, 128-byte swizzle, zero fill behind the last row and the last k), others the
// products and the copies of scales and bias, the rest own the sums.  Every wait on a barrier gives up after some
// seconds and reports QSSM_S_TMA_TIMEOUT; the CTA then still waits for its own copies and products and frees its tensor
// memory.
#pragma once
#include "qssm_elem.cuh"
#include "qssm_tc.cuh"

namespace qssm {

struct MatmulParams {
    CUtensorMap x_map, w_map, y_map;
    const float* x_scales;  // [M, K/128]
    const float* w_scales;  // [N/128, K/128]
    const void* bias;       // [N] or NULL
    void* y;                // [M, N]
    long long xs_row, xs_blk, ws_row, ws_blk, y_stride;
    int M, N, K, n_kb;      // n_kb: blocks of 128 along k
    int m_tiles, n_tiles;
    int bias_dtype, y_vec;  // y_vec: rows of y start on 16-byte boundaries
    int y_word;             // the longest of 8, 4, 2 bytes that every row of y starts and ends on a multiple of
    int* status;
};

constexpr int MM_TIMEOUT = 10001;  // QSSM_S_TMA_TIMEOUT
constexpr int MM_TILE_K = 128;

__device__ __forceinline__ float load_bias(const MatmulParams& p, int n) {
    if (p.bias == nullptr || n >= p.N) return 0.f;
    if (p.bias_dtype == 0) return static_cast<const float*>(p.bias)[n];
    if (p.bias_dtype == 1) return to_f32(static_cast<const __half*>(p.bias)[n]);
    return to_f32(static_cast<const __nv_bfloat16*>(p.bias)[n]);
}
__device__ __forceinline__ float2 as_pair(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }

// ---------------------------------------------------------------------------------------------
// Many rows: two CTAs on neighbouring SMs form 256 x 256 tiles as one product (cta_group::2), each with 128 rows of x,
// half of the weight's 256 rows in shared memory, and the sums of its 128 rows.  Against tiles of 128 x 256 by single
// CTAs that is a third less to read from L2 per product.  Persistent: one pair per two SMs walks the tiles.
//
// Lane = row: a thread owns one row's sums of 128 columns, and both scales of a block are one factor for all of them.
// The product of a block of k is issued as two of 128 columns, each with two buffers of tensor memory of its own.  What
// bounds the kernel is the way of a buffer from its product through both CTAs' sums back to the next product, a chain of
// latencies (issue, commit, test, read back, arrival on the other SM, test; a branch alone is 40 cycles).  So each
// buffer has an issuing warp of its own, and warps of their own fetch the scales (by groups of four blocks) and the next
// tile's bias ahead.  Results leave through shared memory and bulk stores of 32 rows x 128 bytes per warp, so that the
// sums' registers are free for the next tile at once.
//
// 16384x20480x1024 372 us, 1.85 PFLOP/s (429 us under the power limit, 1.54 GHz); 16384x1024x4096 70 us;
// 16384x8192x8192 1.1 ms.  The sums' loop has few branches for the same reason: the next block's scales are read in the
// shadow of the second pair of reads, and the barriers are handed on by predicated arrivals (the warps agreeing on each
// wait's outcome in that loop: 379 us, 72 us).  One product of 256 columns and one issuing warp per block: 391 us (450); one
// issuing warp for all buffers: 438 us; sixteen warps of 64 columns: 426 us.  Tiles of 128 x 256 by single CTAs took 835 us
// in an earlier form whose sums fetched their own scales; they were not measured in this one.
// ---------------------------------------------------------------------------------------------
constexpr int MMR_M = 256, MMR_N = 256, MMR_STAGES = 4;        // a pair's tile
constexpr int MMR_A = 128 * MM_TILE_K, MMR_STAGE = 2 * MMR_A;  // per CTA
constexpr int MMR_WARPS = 8, MMR_COLS = 128;                   // warps that hold sums, columns of each
constexpr int MMR_THREADS = 32 * MMR_WARPS + 256;              // warp 8 copies, 9 to 12 products, 13 scales, 14 bias
// Scales in flight: slots of four blocks, a block being 128 of x and two of w.
constexpr int MMR_SLOTS = 4, MMR_GROUP = 4, MMR_BLOCK = 576, MMR_SLOT = MMR_GROUP * MMR_BLOCK,
              MMR_RING = MMR_SLOTS * MMR_GROUP;
constexpr int MMR_OUT = MMR_STAGES * MMR_STAGE, MMR_BIAS = MMR_OUT + MMR_WARPS * 8192,
              MMR_SCALES = MMR_BIAS + 2 * MMR_N * 4, MMR_BARS = MMR_SCALES + MMR_SLOTS * MMR_SLOT,
              MMR_SMEM = MMR_BARS + 512 + 1024;
// Registers: 128 a thread at launch (512 threads); the eight helper warps give 88 of theirs to the eight others.
constexpr int MMR_REGS_SUMS = 216, MMR_REGS_HELP = 40;
static_assert(256 * MMR_REGS_SUMS + 256 * MMR_REGS_HELP <= MMR_THREADS * 128, "more registers than the CTA has");
static_assert(MMR_SMEM <= 227 * 1024, "more shared memory than a CTA has");

// 32 rows of 128 bytes from shared memory (128-byte swizzle) to `dst`, W bytes a lane.
template <int W>
__device__ __forceinline__ void put_rows(const uint8_t* buf, uint8_t* dst, long long pitch, int rows, int bytes, int lane) {
    constexpr int PER_ROW = 128 / W;  // lanes
    using U = typename Word<W>::type;
#pragma unroll 4
    for (int i = lane; i < 32 * PER_ROW; i += 32) {
        const int r = i / PER_ROW, at = (i % PER_ROW) * W;
        const U v = *reinterpret_cast<const U*>(buf + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15));
        if (r < rows && at < bytes) *reinterpret_cast<U*>(dst + r * pitch + at) = v;
    }
}

template <typename T> __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MMR_THREADS, 1)
    matmul_fp8_rows_kernel(const __grid_constant__ MatmulParams p) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_u32(smem), bars = base + MMR_BARS;
    // full, taken: the even CTA's count for both; the others are each CTA's own.  Buffer b = 2 * (block & 1) + half.
    const uint32_t full = bars, empty = full + 8 * MMR_STAGES, done = empty + 8 * MMR_STAGES, taken = done + 32,
                   scaled = taken + 32, used = scaled + 8 * MMR_SLOTS, biased = used + 8 * MMR_SLOTS,
                   unbiased = biased + 16, last = unbiased + 16;
    static_assert(8 * (2 * MMR_STAGES + 8 + 2 * MMR_SLOTS + 5) + 4 <= 512, "room for the barriers");
    volatile uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + (last + 8 - base));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < MMR_STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 2); }  // empty: both halves
        for (int b = 0; b < 4; ++b) { mbar_init(done + 8 * b, 1); mbar_init(taken + 8 * b, MMR_WARPS); }
        for (int f = 0; f < MMR_SLOTS; ++f) { mbar_init(scaled + 8 * f, 32); mbar_init(used + 8 * f, MMR_WARPS); }
        for (int i = 0; i < 2; ++i) { mbar_init(biased + 8 * i, 1); mbar_init(unbiased + 8 * i, MMR_WARPS); }
        mbar_init(last, 4);
        fence_barrier_init();
    }
    if (warp == MMR_WARPS + 1) tmem_alloc<2>(smem_u32(const_cast<uint32_t*>(tmem_at)), 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_at;
    const int tiles = p.m_tiles * p.n_tiles, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t total = pair < tiles ? (uint32_t)((tiles - pair + pairs - 1) / pairs) * (uint32_t)p.n_kb : 0;
    bool ok = true;

    if (warp >= MMR_WARPS) {
        regs_down<MMR_REGS_HELP>();
        if (warp == MMR_WARPS) {
            const uint32_t full0 = cluster_addr(full, 0);
            uint32_t it = 0;
            for (int t = pair; ok && t < tiles; t += pairs) {
                const int m0 = (t % p.m_tiles) * MMR_M + (int)rank * 128, n0 = (t / p.m_tiles) * MMR_N + (int)rank * 64;
                for (int kb = 0; kb < p.n_kb; ++kb, ++it) {
                    const uint32_t s = it % MMR_STAGES, round = it / MMR_STAGES;
                    if (round > 0) ok = mbar_wait_limit(empty + 8 * s, (round - 1) & 1);
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                    if (elect_one()) {
                        const uint32_t at = base + s * MMR_STAGE, bar = full0 + 8 * s;
                        if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * MMR_STAGE);
                        tma_load_2d_pair(at, &p.x_map, bar, kb * MM_TILE_K, m0);
                        tma_load_2d_pair(at + MMR_A, &p.w_map, bar, kb * MM_TILE_K, n0);
                        tma_load_2d_pair(at + MMR_A + MMR_A / 2, &p.w_map, bar, kb * MM_TILE_K, n0 + 128);
                    }
                }
            }
            // no copy outlives the pair: the last rounds' products are done (both CTAs are told), or time is given
            const uint32_t left = it < (uint32_t)MMR_STAGES ? it : (uint32_t)MMR_STAGES;
            for (uint32_t i = it - left; ok && i < it; ++i) ok = mbar_wait_limit(empty + 8 * (i % MMR_STAGES), (i / MMR_STAGES) & 1);
            if (!ok) wait_ns(1000000);
        } else if (warp <= MMR_WARPS + 4) {
            if (rank == 0) {  // warp 9 + b issues the products of buffer b: every second block's, of one half of the columns
                constexpr uint32_t idesc = fp8_idesc(MMR_M, 128);
                const uint32_t b = warp - (MMR_WARPS + 1), half = b & 1;
                const uint32_t my_taken = taken + 8 * b, my_done = done + 8 * b, d = tmem + b * 128;
                uint32_t round = 0;
                for (uint32_t it = b >> 1; it < total; it += 2, ++round) {
                    const uint32_t s = it % MMR_STAGES;
                    const uint64_t x = smem_operand(base + s * MMR_STAGE),
                                   w = smem_operand(base + s * MMR_STAGE + MMR_A + half * (MMR_A / 2));
                    ok = mbar_wait_limit(full + 8 * s, (it / MMR_STAGES) & 1);
                    if (round > 0) ok &= mbar_wait_limit(my_taken, (round - 1) & 1);
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) tc_mma_fp8_pair(d, x + 2 * k, w + 2 * k, idesc, k > 0);
                        tc_commit_pair(my_done);
                        tc_commit_pair(empty + 8 * s);
                    }
                    __syncwarp();
                }
                if (elect_one()) tc_commit_group2(last);  // no product outlives the pair
                ok &= mbar_wait_limit(last, 0);
                // nor an arrival from the other CTA: it would land in the barriers of the next kernel on this SM
                if (round > 0) ok &= mbar_wait_limit(my_taken, (round - 1) & 1);
            }
        } else if (warp == MMR_WARPS + 5) {
            uint32_t it = 0;
            for (int t = pair; ok && t < tiles; t += pairs) {
                const int m0 = (t % p.m_tiles) * MMR_M + (int)rank * 128 + lane, n0 = (t / p.m_tiles) * MMR_N + (lane & 1) * 128;
                const float* w = p.w_scales + (long long)(n0 < p.N ? n0 / 128 : 0) * p.ws_row;
                const float* xs[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) xs[i] = p.x_scales + (long long)(m0 + 32 * i < p.M ? m0 + 32 * i : 0) * p.xs_row;
                for (int kb = 0; kb < p.n_kb; ++kb, ++it) {
                    const uint32_t group = it / MMR_GROUP, f = group % MMR_SLOTS, round = group / MMR_SLOTS;
                    if (it % MMR_GROUP == 0 && round > 0) ok = mbar_wait_limit(used + 8 * f, (round - 1) & 1);
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                    const uint32_t at = base + MMR_SCALES + it % MMR_RING * MMR_BLOCK + lane * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        copy_4(at + 128 * i, xs[i]);
                        xs[i] += p.xs_blk;
                    }
                    if (lane < 2) copy_4(at + 512, w);
                    w += p.ws_blk;
                    if (it % MMR_GROUP == MMR_GROUP - 1 || it + 1 == total) copies_arrive(scaled + 8 * f);
                }
            }
            copies_wait();
        } else if (warp == MMR_WARPS + 6 && p.bias != nullptr) {  // the next tile's bias while this one is worked on
            uint32_t turn = 0;
            for (int t = pair; ok && t < tiles; t += pairs, ++turn) {
                const int n0 = (t / p.m_tiles) * MMR_N;
                float v[MMR_N / 32];
#pragma unroll
                for (int i = 0; i < MMR_N / 32; ++i) v[i] = load_bias(p, n0 + 32 * i + lane);
                if (turn >= 2) ok = mbar_wait_limit(unbiased + 8 * (turn & 1), ((turn >> 1) - 1) & 1);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                float* to = reinterpret_cast<float*>(smem + MMR_BIAS) + (turn & 1) * MMR_N;
#pragma unroll
                for (int i = 0; i < MMR_N / 32; ++i) to[32 * i + lane] = v[i];
                __syncwarp();
                if (lane == 0) mbar_arrive(biased + 8 * (turn & 1));
            }
        }
    } else {
        regs_up<MMR_REGS_SUMS>();
        const int quarter = warp & 3, half = warp >> 2, col0 = half * MMR_COLS;
        const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16) + half * 128;
        const uint32_t taken0 = cluster_addr(taken, 0) + 8 * half, my_done = done + 8 * half;
        const float* my_x = reinterpret_cast<const float*>(smem + MMR_SCALES) + quarter * 32 + lane;
        const float* my_w = reinterpret_cast<const float*>(smem + MMR_SCALES) + 128 + half;
        auto scales_here = [&](uint32_t i) {
            return mbar_wait_limit(scaled + 8 * (i / MMR_GROUP % MMR_SLOTS), (i / MMR_RING) & 1);
        };
        uint32_t it = 0, turn = 0;
        if (total > 0) ok = scales_here(0);
        float sx = my_x[0], sw = my_w[0];  // the next block's
        for (int t = pair; ok && t < tiles; t += pairs, ++turn) {
            const int m0 = (t % p.m_tiles) * MMR_M + (int)rank * 128 + quarter * 32, n0 = (t / p.m_tiles) * MMR_N + col0;
            float2 acc[MMR_COLS / 2];
            if (p.bias != nullptr) {  // the sums start from the bias
                ok = mbar_wait_limit(biased + 8 * (turn & 1), (turn >> 1) & 1);
                const float* bias = reinterpret_cast<const float*>(smem + MMR_BIAS) + (turn & 1) * MMR_N + col0;
#pragma unroll
                for (int j = 0; j < MMR_COLS / 4; ++j) {
                    const float4 v = *reinterpret_cast<const float4*>(bias + 4 * j);
                    acc[2 * j] = make_float2(v.x, v.y);
                    acc[2 * j + 1] = make_float2(v.z, v.w);
                }
                __syncwarp();
                mbar_arrive_if(lane == 0 && ok, unbiased + 8 * (turn & 1));
            } else {
                __syncwarp();  // one lane stored the tile before: the loop's loads are the whole warp's
#pragma unroll
                for (int j = 0; j < MMR_COLS / 2; ++j) acc[j] = make_float2(0.f, 0.f);
            }
            for (int kb = 0; ok && kb < p.n_kb; ++kb, ++it) {
                const uint32_t b = it & 1, d = at + b * 256, ni = it + 1;
                ok &= mbar_wait_limit(my_done + 16 * b, (it >> 1) & 1);
                tc_fence_after();
                uint32_t r0[32], r1[32];
                tmem_ld<32>(d, r0);
                tmem_ld<32>(d + 32, r1);
                const float factor = sx * sw;  // scale of the row x scale of the weight's block
                const float2 s = make_float2(factor, factor);
                tc_wait_ld(r0);
                tc_landed(r1);
#pragma unroll
                for (int j = 0; j < 16; ++j) fma_pair(acc[j], as_pair(r0[2 * j], r0[2 * j + 1]), s);
                tmem_ld<32>(d + 64, r0);
#pragma unroll
                for (int j = 0; j < 16; ++j) fma_pair(acc[16 + j], as_pair(r1[2 * j], r1[2 * j + 1]), s);
                tmem_ld<32>(d + 96, r1);
                // while those come: the next block's scales
                if (ni % MMR_GROUP == 0 && ni < total) ok &= scales_here(ni);
                sx = my_x[ni % MMR_RING * (MMR_BLOCK / 4)];
                sw = my_w[ni % MMR_RING * (MMR_BLOCK / 4)];
                tc_wait_ld(r0);
                tc_landed(r1);
                tc_fence_before();  // all read: the buffer may be written again
                mbar_arrive_cluster_if(lane == 0 && ok, taken0 + 16 * b);
                mbar_arrive_if(lane == 0 && ok && ni % MMR_GROUP == 0, used + 8 * (it / MMR_GROUP % MMR_SLOTS));
#pragma unroll
                for (int j = 0; j < 16; ++j) fma_pair(acc[32 + j], as_pair(r0[2 * j], r0[2 * j + 1]), s);
#pragma unroll
                for (int j = 0; j < 16; ++j) fma_pair(acc[48 + j], as_pair(r1[2 * j], r1[2 * j + 1]), s);
            }
            if (!ok || m0 >= p.M || n0 >= p.N) continue;
            // 128 bytes of each row at a time; 16-byte piece c of row r lies at c ^ (r & 7), where a bulk store in the
            // 128-byte swizzle looks for it, and eight lanes' pieces in eight different banks
            constexpr int V = 16 / sizeof(T), COLS = 8 * V, CHUNKS = MMR_COLS / COLS;
            uint8_t* const bufs = smem + MMR_OUT + warp * 8192;
#pragma unroll
            for (int c0 = 0; c0 < CHUNKS; c0 += 2) {  // two pieces behind one fence
                if (lane == 0) tma_wait_read<0>();  // the stores that read these buffers before
                __syncwarp();
#pragma unroll
                for (int c = c0; c < c0 + 2; ++c)
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        float v[V];
#pragma unroll
                        for (int i = 0; i < V; i += 2) {
                            v[i] = acc[(c * COLS + q * V + i) / 2].x;
                            v[i + 1] = acc[(c * COLS + q * V + i) / 2].y;
                        }
                        store_elems<T, V>(reinterpret_cast<T*>(bufs + (c - c0) * 4096 + lane * 128 + ((q ^ (lane & 7)) << 4)), v);
                    }
                if (p.y_vec) {
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        if (n0 + c0 * COLS < p.N) tma_store_2d(&p.y_map, smem_u32(bufs), n0 + c0 * COLS, m0);
                        if (n0 + (c0 + 1) * COLS < p.N) tma_store_2d(&p.y_map, smem_u32(bufs) + 4096, n0 + (c0 + 1) * COLS, m0);
                        tma_commit();
                    }
                } else {  // rows of y on any boundary: each row's 128 bytes by consecutive lanes, in the words that fit
                    __syncwarp();
                    const int rows = p.M - m0 < 32 ? p.M - m0 : 32;
                    const long long pitch = p.y_stride * sizeof(T);
#pragma unroll
                    for (int c = c0; c < c0 + 2; ++c) {
                        const int bytes = (p.N - n0 - c * COLS) * (int)sizeof(T);
                        const uint8_t* buf = bufs + (c - c0) * 4096;
                        uint8_t* dst = static_cast<uint8_t*>(p.y) + ((long long)m0 * p.y_stride + n0 + c * COLS) * sizeof(T);
                        if (p.y_word == 8) put_rows<8>(buf, dst, pitch, rows, bytes, lane);
                        else if (p.y_word == 4) put_rows<4>(buf, dst, pitch, rows, bytes, lane);
                        else put_rows<2>(buf, dst, pitch, rows, bytes, lane);
                    }
                }
            }
        }
        if (lane == 0) tma_wait_all();
    }
    if (!ok && lane == 0 && p.status != nullptr) *p.status = MM_TIMEOUT;
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    if (warp == MMR_WARPS + 1) tmem_free<2>(tmem, 512);
}

// ---------------------------------------------------------------------------------------------
// Few rows: the weight is the first operand.  Tiles of 128 columns of y x T rows (T = 16 to 128), lane = column, so
// the weight's rows fill the tensor cores' 128 lanes however few rows there are, and k is cut over the S CTAs of a
// cluster, whose sums are added in rank order through distributed shared memory (each CTA adds every S-th row).
// Bound by latencies: a CTA sees few blocks of k, each a copy, a product and a read back, behind some 4 us of launch and
// set-up.  1x20480x1024 7.1 us (160 CTAs of eight blocks, k not cut), 64x1024x4096 7.6 us (64 CTAs of four blocks and the
// join); the many-rows kernel 14.4 and 18.9.
// ---------------------------------------------------------------------------------------------
template <int T> struct Few {
    static constexpr int A = 128 * MM_TILE_K, STAGE = A + T * MM_TILE_K;
    static constexpr int PER_SM = T <= 64 ? 2 : 1;                  // CTAs on an SM
    static constexpr int STAGES = T <= 32 ? 5 : T == 64 ? 4 : 6;
    static constexpr int BUFS = T <= 64 ? 4 : 2;
    static constexpr uint32_t TMEM = BUFS * T;                      // 64 to 256 columns
    static constexpr int WARPS = T <= 64 ? 4 : 8;                   // warps that hold sums, each of 32 columns x ROWS rows
    static constexpr int ROWS = 4 * T / WARPS;
    static constexpr int THREADS = 32 * WARPS + 96;                 // then a warp each for copies, products, scales
    static constexpr int SLOTS = 8, SLOT = 4 * (T + 4);             // blocks of scales in flight: T of x, one of w
    static constexpr int SCALES = STAGES * STAGE, BARS = SCALES + SLOTS * SLOT, SMEM = BARS + 512 + 1024;
    static_assert(8 * (2 * STAGES + 2 * BUFS + 2 * SLOTS + 1) + 4 <= 512, "room for the barriers");
    static_assert(PER_SM * (SMEM + 1024) <= 228 * 1024, "more shared memory than an SM has");
    static_assert(STAGES * STAGE >= T * 128 * 4, "the sums are handed over in the stages' memory");
};

template <typename OUT, int T>
__global__ void __launch_bounds__(Few<T>::THREADS, Few<T>::PER_SM) matmul_fp8_few_kernel(const __grid_constant__ MatmulParams p, int S) {
    using C = Few<T>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_u32(smem), full = base + C::BARS;
    const uint32_t empty = full + 8 * C::STAGES, done = empty + 8 * C::STAGES, taken = done + 8 * C::BUFS,
                   scaled = taken + 8 * C::BUFS, used = scaled + 8 * C::SLOTS, last = used + 8 * C::SLOTS;
    volatile uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + (last + 8 - base));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (int b = 0; b < C::BUFS; ++b) { mbar_init(done + 8 * b, 1); mbar_init(taken + 8 * b, C::WARPS); }
        for (int f = 0; f < C::SLOTS; ++f) { mbar_init(scaled + 8 * f, 32); mbar_init(used + 8 * f, C::WARPS); }
        mbar_init(last, 1);
        fence_barrier_init();
    }
    if (warp == C::WARPS + 1) tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_at)), C::TMEM);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_at;
    const int rank = S > 1 ? (int)cluster_rank() : 0;
    const int n0 = ((int)blockIdx.x / S) * 128, m0 = (int)blockIdx.y * T;
    const int kb0 = (int)((long long)p.n_kb * rank / S), blocks = (int)((long long)p.n_kb * (rank + 1) / S) - kb0;
    const int n = n0 + (warp & 3) * 32 + lane, row0 = (warp >> 2) * C::ROWS;  // of the warps with sums
    float2 acc[C::ROWS / 2];
    bool ok = true;

    if (warp == C::WARPS) {
        for (int it = 0; it < blocks; ++it) {
            const int s = it % C::STAGES, round = it / C::STAGES;
            if (round > 0) ok = mbar_wait_limit(empty + 8 * s, (round - 1) & 1);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            if (elect_one()) {
                mbar_expect_tx(full + 8 * s, C::STAGE);
                tma_load_2d(base + s * C::STAGE, &p.w_map, full + 8 * s, (kb0 + it) * MM_TILE_K, n0);
                tma_load_2d(base + s * C::STAGE + C::A, &p.x_map, full + 8 * s, (kb0 + it) * MM_TILE_K, m0);
            }
        }
        // no copy outlives the CTA: the last rounds' products are done, or time is given
        for (int i = blocks < C::STAGES ? 0 : blocks - C::STAGES; ok && i < blocks; ++i)
            ok = mbar_wait_limit(empty + 8 * (i % C::STAGES), (i / C::STAGES) & 1);
        if (!ok) wait_ns(1000000);
    } else if (warp == C::WARPS + 1) {
        constexpr uint32_t idesc = fp8_idesc(128, T);
        for (int it = 0; it < blocks; ++it) {
            const int s = it % C::STAGES, b = it % C::BUFS, round = it / C::BUFS;
            const uint64_t w = smem_operand(base + s * C::STAGE), x = smem_operand(base + s * C::STAGE + C::A);
            ok = mbar_wait_limit(full + 8 * s, (it / C::STAGES) & 1);
            if (round > 0) ok &= mbar_wait_limit(taken + 8 * b, (round - 1) & 1);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_fp8(tmem + b * T, w + 2 * k, x + 2 * k, idesc, k > 0);
                tc_commit(done + 8 * b);
                tc_commit(empty + 8 * s);
            }
            __syncwarp();
        }
        if (elect_one()) tc_commit(last);  // no product outlives the CTA
        ok &= mbar_wait_limit(last, 0);
    } else if (warp == C::WARPS + 2) {
        constexpr int PER = (T + 31) / 32;
        const float* ws = p.w_scales + (long long)(n0 / 128) * p.ws_row + kb0 * p.ws_blk;
        const float* xs[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int m = m0 + i * 32 + lane;
            xs[i] = p.x_scales + (long long)(m < p.M ? m : 0) * p.xs_row + kb0 * p.xs_blk;
        }
        for (int it = 0; it < blocks; ++it) {
            const int f = it % C::SLOTS, round = it / C::SLOTS;
            if (round > 0) ok = mbar_wait_limit(used + 8 * f, (round - 1) & 1);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            const uint32_t at = base + C::SCALES + f * C::SLOT;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (i * 32 + lane < T) copy_4(at + (i * 32 + lane) * 4, xs[i]);
                xs[i] += p.xs_blk;
            }
            if (lane == 0) copy_4(at + T * 4, ws);
            ws += p.ws_blk;
            copies_arrive(scaled + 8 * f);
        }
        copies_wait();
    } else {
#pragma unroll
        for (int j = 0; j < C::ROWS / 2; ++j) acc[j] = make_float2(0.f, 0.f);
        const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + row0;
        for (int it = 0; ok && it < blocks; ++it) {
            const int f = it % C::SLOTS, b = it % C::BUFS;
            const float* scale = reinterpret_cast<const float*>(smem + C::SCALES + f * C::SLOT);
            ok = mbar_wait_limit(scaled + 8 * f, (it / C::SLOTS) & 1);
            const float sw = scale[T];
            ok &= mbar_wait_limit(done + 8 * b, (it / C::BUFS) & 1);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;  // what follows is the whole warp's
            tc_fence_after();
            constexpr int L = C::ROWS < 32 ? C::ROWS : 32;  // rows read back at a time
#pragma unroll
            for (int c = 0; c < C::ROWS / L; ++c) {
                uint32_t r[L];
                tmem_ld<L>(at + b * T + c * L, r);
                tc_wait_ld(r);
                if (c + 1 == C::ROWS / L) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0 && ok) mbar_arrive(taken + 8 * b);
                }
#pragma unroll
                for (int j = 0; j < L / 4; ++j) {
                    const float4 s = *reinterpret_cast<const float4*>(scale + row0 + c * L + 4 * j);
                    fma_pair(acc[c * L / 2 + 2 * j], as_pair(r[4 * j], r[4 * j + 1]), make_float2(s.x * sw, s.y * sw));
                    fma_pair(acc[c * L / 2 + 2 * j + 1], as_pair(r[4 * j + 2], r[4 * j + 3]), make_float2(s.z * sw, s.w * sw));
                }
            }
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(used + 8 * f);
        }
    }
    if (!ok && lane == 0 && p.status != nullptr) *p.status = MM_TIMEOUT;
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == C::WARPS + 1) tmem_free<1>(tmem, C::TMEM);
    if (S > 1) {
        float* sums = reinterpret_cast<float*>(smem);  // [T][128]
        if (warp < C::WARPS) {
#pragma unroll
            for (int j = 0; j < C::ROWS / 2; ++j) {
                sums[(row0 + 2 * j) * 128 + (warp & 3) * 32 + lane] = acc[j].x;
                sums[(row0 + 2 * j + 1) * 128 + (warp & 3) * 32 + lane] = acc[j].y;
            }
        }
        cluster_sync();
        if (warp < C::WARPS && n < p.N) {
            const float bias = load_bias(p, n);
            // four rows' partial sums on their way at once: a load from another SM takes longer than anything here
            const int step = S * (C::WARPS / 4), rows = p.M - m0 < T ? p.M - m0 : T;
            for (int j0 = rank + (warp >> 2) * S; j0 < rows; j0 += 4 * step) {
                float v[4][8];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int j = j0 + i * step;
                        v[i][q] = q < S && j < rows ? ld_cluster(base + (uint32_t)(j * 128 + (warp & 3) * 32 + lane) * 4u, q) : 0.f;
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + i * step;
                    float sum = bias;
#pragma unroll
                    for (int q = 0; q < 8; ++q) sum += v[i][q];
                    if (j < rows) static_cast<OUT*>(p.y)[(long long)(m0 + j) * p.y_stride + n] = from_f32<OUT>(sum);
                }
            }
        }
        cluster_sync();  // no CTA leaves while its sums may be read
    } else if (warp < C::WARPS && n < p.N) {
        const float bias = load_bias(p, n);
        OUT* y = static_cast<OUT*>(p.y) + (long long)(m0 + row0) * p.y_stride + n;
#pragma unroll
        for (int j = 0; j < C::ROWS; ++j)
            if (m0 + row0 + j < p.M) y[j * p.y_stride] = from_f32<OUT>(bias + (j & 1 ? acc[j / 2].y : acc[j / 2].x));
    }
}

}  // namespace qssm
