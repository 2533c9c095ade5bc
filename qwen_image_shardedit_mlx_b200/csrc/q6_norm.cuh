// Layer norm over rows of D, forward and gradients (q6_layer_norm,
// q6_layer_norm_grad):
//   y = xh w + b,  xh = (x - mean) rstd
//   a = dy w,  dx = rstd (a - mean_D(a) - xh mean_D(a xh)),
//   dweight = sum over rows of dy xh,  dbias = sum over rows of dy.
// Statistics and sums in fp32 (the variance from centred values, a second
// pass over registers); one rounding at each output.
//
// Both directions are bound by HBM: the forward reads x and writes y, the
// backward reads x and dy and writes dx, once each: the forward holds a row in
// the registers of one thread group of W warps, the backward a tile of rows in
// shared memory.  In the backward a thread keeps the same columns for every row
// it sees, so the weight's and bias's gradients accumulate in registers over a
// strip of rows; a CTA adds its thread groups in order, and a second kernel adds
// the strips' sums in order.  No atomics: equal calls give equal bits.
//
// Each thread holds N groups of G elements (16 bytes).  Where D, strides and
// addresses allow it a group is one 16-byte access; else its G elements lie a
// thread group apart (one access each, neighbouring threads on neighbouring
// elements).  Rows too wide for registers take plain kernels (q6_norm.cu: one
// CTA per row, several passes).
#pragma once

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <iterator>
#include <type_traits>
#include <utility>

#include "q6_dense.cuh"
#include "q6_internal.h"
#include "q6_ptx.cuh"

namespace q6 {

constexpr int64_t kNormMaxGrid = (int64_t(1) << 31) - 1;

struct NormParams {
    const void* x;
    int64_t ldx;
    const void* weight;
    const void* bias;
    int64_t ldv, rows_per_vec;
    void* y;
    float* mean;
    float* rstd;
    int64_t M, D;
    float eps;
    float one;  // added to the weight: 1 with Q6_NORM_ONE_PLUS
    // gradients
    const void* dy;
    int64_t ldy;
    void* dx;
    float* dw_part;  // [strips, D] or null
    float* db_part;
    int64_t strip_rows, strips_per_vec;
    unsigned col_blocks;
    unsigned vecs;  // forward: vectors, where they are the grid's second axis (else 0)
    float inv, inv_rest;  // forward: 1 / D rounded, and what the rounding left
};


namespace norm_detail {

// Sum over the 32 lanes of each of v's two values, in every lane: the first
// exchange leaves one value per lane, so two sums cost six shuffles.
__device__ __forceinline__ float2 warp_sum2(float2 v) {
    const bool odd = threadIdx.x & 1;
    float s = odd ? v.y : v.x;
    s += __shfl_xor_sync(0xffffffffu, odd ? v.x : v.y, 1);
#pragma unroll
    for (int o = 2; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float other = __shfl_xor_sync(0xffffffffu, s, 1);
    return odd ? make_float2(other, s) : make_float2(s, other);
}

// The mean of a row from its sum, rounded once: sum (inv + inv_rest) carries 1 / D to 47
// bits.  sum * inv alone may be a step off; for a constant row (padding) the variance
// takes that step for the row's spread, and 1920 values of -65504 came out as +-1.
// An infinite sum stays so.  (A division costs registers: 5000 x 12288 40.6 -> 52.9 us.)
__device__ __forceinline__ float norm_mean(float sum, const NormParams& p) {
    const float rest = __fmul_rn(sum, p.inv_rest);
    return __fmaf_rn(sum, p.inv, isinf(sum) ? 0.0f : rest);
}

// Sum over each run of L lanes.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// How a thread group's accesses lie: one element at a time, 16 bytes at a time,
// or 16 bytes at a time with every group of every thread inside the row (no
// bounds to test: they were a third of the instructions).
enum Layout { kStrided = 0, kVec = 1, kFull = 2 };

// Which columns a thread holds: group j of G elements of thread t of a group of
// `threads`, either contiguous or a thread group apart.
template <typename T, Layout kLay, int kThreads>
struct Columns {
    static constexpr int G = 16 / sizeof(T);
    int t, D;
    __device__ __forceinline__ int column(int j, int i) const {
        return kLay != kStrided ? (t + kThreads * j) * G + i : t + kThreads * (j * G + i);
    }
    // the slot (j * G + i) and the thread that hold column c
    static __device__ __forceinline__ int slot(int c) {
        return kLay != kStrided ? c / (G * kThreads) * G + c % G : c / kThreads;
    }
    static __device__ __forceinline__ int thread(int c) {
        return kLay != kStrided ? c / G % kThreads : c % kThreads;
    }
    // any column of group j is inside the row
    __device__ __forceinline__ bool some(int j) const { return kLay == kFull || column(j, 0) < D; }
    // element i of group j is; a contiguous group is inside or outside as a whole
    __device__ __forceinline__ bool inside(int j, int i) const { return kLay != kStrided || column(j, i) < D; }

    // Group j of a row of S.  Strided: elements outside the row are zero;
    // contiguous groups outside it are not defined.
    template <typename S>
    __device__ __forceinline__ Group<S, G> load(const S* row, int j) const {
        Group<S, G> g;
        if constexpr (kLay != kStrided) {
            if (some(j)) g = load_ro<Group<S, G>>(row + column(j, 0));
        } else {
#pragma unroll
            for (int i = 0; i < G; ++i) g.v[i] = inside(j, i) ? load_ro<S>(row + column(j, i)) : from_f<S>(0.0f);
        }
        return g;
    }
    template <typename S>
    __device__ __forceinline__ void store(S* row, int j, const Group<S, G>& g) const {
        if constexpr (kLay != kStrided) {
            if (some(j)) *reinterpret_cast<Group<S, G>*>(row + column(j, 0)) = g;
        } else {
#pragma unroll
            for (int i = 0; i < G; ++i)
                if (inside(j, i)) row[column(j, i)] = g.v[i];
        }
    }
    // The factor one + w of group j (1 without a weight).
    template <typename S>
    __device__ __forceinline__ void factor(const S* w, int j, float one, float2 (&f)[G / 2]) const {
        if (w) {
            unpack(load(w, j), f);
#pragma unroll
            for (int i = 0; i < G / 2; ++i) f[i] = add2(f[i], both(one));
        } else {
#pragma unroll
            for (int i = 0; i < G / 2; ++i) f[i] = both(1.0f);
        }
    }
};

// Forward: W warps per row (one row per CTA), or L lanes (128 / L rows per CTA; a
// row of 128 in a warp of its own left half its lanes idle: 165888 rows of bf16
// 37.6 us, 20.8 so), N groups per thread.  N is at most four: a row's code runs
// once per row, and with twelve groups per lane (a warp per row of 3072) its
// unrolled length ran out of the instruction cache: 31 us for 6912 rows of bf16
// against 21 us with four.  The grid is one wave of CTAs that walk the rows, the
// next row's loads in flight while a row is summed: 15.5 us (5.5 TB/s).
template <typename T, typename V, Layout kLay, int W, int N, int L>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W) norm_kernel(const NormParams p) {
    constexpr int G = 16 / sizeof(T), kRows = W == 1 ? 128 / L : 1;
    static_assert(L == 32 || W == 1, "lanes of one warp");
    __shared__ float parts[2][W];
    pdl_launch_dependents();
    // rows first, first + step, ... of a vector's rows, or of all where the vectors are not the grid's second axis
    const int64_t limit = p.vecs ? p.rows_per_vec : p.M, step = gridDim.x * int64_t(kRows);
    int64_t local = W == 1 ? blockIdx.x * int64_t(kRows) + threadIdx.x / L : int64_t(blockIdx.x);
    int64_t warp_row = W == 1 ? blockIdx.x * int64_t(kRows) + threadIdx.x / 32 * (32 / L) : int64_t(blockIdx.x);
    if (warp_row >= limit) return;  // a whole warp
    // lanes past the last row follow their warp on that row, and store nothing
    auto row_of = [&](int64_t r) { return L < 32 ? min(r, limit - 1) : r; };
    const int64_t row0 = p.vecs ? blockIdx.y * p.rows_per_vec : 0;
    pdl_wait();
    const Columns<T, kLay, L * W> at{W == 1 ? static_cast<int>(threadIdx.x % L) : static_cast<int>(threadIdx.x),
                                     static_cast<int>(p.D)};
    auto row_sum = [&](float v, int flip) {
        v = lanes_sum<L>(v);
        if constexpr (W > 1) {
            if ((at.t & 31) == 0) parts[flip][at.t >> 5] = v;
            __syncthreads();
            v = parts[flip][0];
#pragma unroll
            for (int i = 1; i < W; ++i) v += parts[flip][i];
        }
        return v;
    };
    const T* x = static_cast<const T*>(p.x) + (row0 + row_of(local)) * p.ldx;
    Group<T, G> in[N];
#pragma unroll
    for (int j = 0; j < N; ++j) in[j] = at.load(x, j);
    for (;; local += step, warp_row += step) {
        const int64_t row = row0 + row_of(local);
        const bool more = warp_row + step < limit, ours = L == 32 || local < limit;
        Group<T, G> next[N];
        if (more) {
            if constexpr (L == 32)
                x += step * p.ldx;
            else
                x = static_cast<const T*>(p.x) + (row0 + row_of(local + step)) * p.ldx;
#pragma unroll
            for (int j = 0; j < N; ++j) next[j] = at.load(x, j);
        }
        int64_t v0 = 0;
        if (p.vecs)
            v0 = blockIdx.y * p.ldv;
        else if (p.rows_per_vec < p.M)
            v0 = row / p.rows_per_vec * p.ldv;
        const V* w = p.weight ? static_cast<const V*>(p.weight) + v0 : nullptr;
        const V* b = p.bias ? static_cast<const V*>(p.bias) + v0 : nullptr;
        float2 c[N][G / 2];
        float2 s = both(0.0f);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (at.some(j)) {
                unpack(in[j], c[j]);
#pragma unroll
                for (int i = 0; i < G / 2; ++i) s = add2(s, c[j][i]);
            }
        }
        const float mean = norm_mean(row_sum(s.x + s.y, 0), p);
        float2 q = both(0.0f);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (at.some(j)) {
#pragma unroll
                for (int i = 0; i < G / 2; ++i) {
                    c[j][i] = add2(c[j][i], both(-mean));
                    if constexpr (kLay == kStrided) {
                        if (!at.inside(j, 2 * i)) c[j][i].x = 0.0f;
                        if (!at.inside(j, 2 * i + 1)) c[j][i].y = 0.0f;
                    }
                    q = fma2(c[j][i], c[j][i], q);
                }
            }
        }
        const float rstd = rsqrtf(row_sum(q.x + q.y, 1) * p.inv + p.eps);
        if (p.mean && at.t == 0 && ours) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
        T* y = static_cast<T*>(p.y) + row * p.D;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (ours && at.some(j)) {
                float2 fw[G / 2], fb[G / 2];
                at.factor(w, j, p.one, fw);
#pragma unroll
                for (int i = 0; i < G / 2; ++i) fb[i] = both(0.0f);
                if (b) unpack(at.load(b, j), fb);
#pragma unroll
                for (int i = 0; i < G / 2; ++i) fb[i] = fma2(mul2(c[j][i], both(rstd)), fw[i], fb[i]);
                at.store(y, j, pack<T, G>(fb));
            }
        }
        if (!more) return;
#pragma unroll
        for (int j = 0; j < N; ++j) in[j] = next[j];
    }
}

// Makes the compiler forget what it derived from a group's registers.
template <typename T, int G>
__device__ __forceinline__ void keep_packed(Group<T, G>& g) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&g);
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+r"(w[i]));
}

// The column sums of a CTA's RL row lanes of kThreads threads each, added in row
// lane order, to the strip's partial sums or to the result.  sums: finish_bytes()
// of shared memory that nobody reads any more after the first barrier; a slot
// (one of a thread's values) per row of kThreads words padded by four, so that
// writing by thread and reading by column both hit distinct banks.
template <int RL, int kThreads, int N, int G>
constexpr size_t finish_bytes() {
    return size_t(RL) * (kThreads + 4) * 2 * N * G * sizeof(float);
}

template <int RL, int kThreads, typename C, typename V, int N, int P>
__device__ __forceinline__ void finish_columns(const NormParams& p, const C& at, int row_lane, int64_t strip, float* sums,
                                               const float2 (&dw)[N][P], const float2 (&db)[N][P], V* dweight, V* dbias) {
    constexpr int kSlots = 2 * N * P, kRow = kThreads + 4;  // slots of dw; as many of db follow
    __syncthreads();
    float* mine = sums + row_lane * (2 * kSlots * kRow) + at.t;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const int slot = (j * P + e) * 2;
            mine[slot * kRow] = dw[j][e].x;
            mine[(slot + 1) * kRow] = dw[j][e].y;
            mine[(kSlots + slot) * kRow] = db[j][e].x;
            mine[(kSlots + slot + 1) * kRow] = db[j][e].y;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < at.D; c += RL * kThreads) {
        const float* from = sums + C::slot(c) * kRow + C::thread(c);
        float w = 0.0f, b = 0.0f;
#pragma unroll
        for (int r = 0; r < RL; ++r) {
            w += from[r * (2 * kSlots * kRow)];
            b += from[r * (2 * kSlots * kRow) + kSlots * kRow];
        }
        const int64_t to = strip * p.D + c;
        if (p.dw_part) p.dw_part[to] = w;
        if (p.db_part) p.db_part[to] = b;
        if (dweight) dweight[to] = from_f<V>(w);
        if (dbias) dbias[to] = from_f<V>(b);
    }
}

// Backward.  A CTA takes one strip of rows (all of one vector) in tiles of
// TR = RL * M rows, in two phases with one barrier between them:
//   A  every row of the tile is summed by CW / M warps (sum a, sum a xh);
//   B  every thread keeps N groups of columns (CW warps cover the row, RL row
//      lanes side by side) for M rows of the tile: dx, and the column sums of
//      dy xh and dy in registers.
// Tiles arrive by bulk copies in a ring of stages.  The thread that refills a
// stage does so after the barrier of the next tile, which every thread passes
// after its last read of the stage.  With x and dy held in registers and a
// barrier per row instead, 6912 rows of 3072 took 46 us: a row's chain of
// shuffles, barrier and sums left the SM idle.
//   In B: dx = rstd (dy w + xh k + c),  k = -mean_D(a xh),  c = -mean_D(a);  dweight += dy xh.
// Both phases form xh = (x - mean) rstd before anything is multiplied with it, and rstd
// enters dx last: every intermediate value then has the scale of an input or output.  (With
// sums of a (x - mean) and a coefficient rstd^2 mean_D(a xh) a multiply per pair of values
// is saved, but rstd^3 leaves fp32 on the way: rows of a standard deviation from 1e13 on
// lost the third term, rows of 1e-14 with eps = 0 gave infinities.)
// Row lanes: about 384 threads.  Fewer threads mean smaller tiles, so more of
// them in flight: with 576, two stages of 72 KB, a tile's copy had half a tile's
// time to land (65536 x 1024 fp16 110 us, 80 so; 256 threads 96).
constexpr int grad_row_lanes(int cw) { return 12 / cw < 1 ? 1 : 12 / cw; }
constexpr int kGradSmem = 208 * 1024;
constexpr int kGradMaxStages = 8;

template <typename T, typename V, Layout kLay, int CW, int N, int M>
__global__ void __launch_bounds__(32 * CW * grad_row_lanes(CW), 1)
    norm_grad_kernel(const NormParams p, V* dweight, V* dbias, const int stages) {
    constexpr int G = 16 / sizeof(T), P = G / 2, RL = grad_row_lanes(CW), TR = RL * M;
    constexpr int AP = CW >= M ? CW / M : 1, AR = CW >= M ? 1 : M / CW;  // warps per row and rows per warp in phase A
    static_assert((CW >= M ? CW % M : M % CW) == 0 && kLay != kStrided, "phase A");
    __shared__ __align__(16) float2 parts[2][TR][AP];
    __shared__ float4 stats[2][TR];  // -mean, rstd and, with a warp per row in phase A, c and k
    __shared__ __align__(8) uint64_t full[kGradMaxStages];
    __shared__ int abort_word;
    extern __shared__ __align__(128) uint8_t smem[];  // the ring, the factors [D]; in the end the column sums (finish_bytes)
    pdl_launch_dependents();
    const int D = static_cast<int>(p.D), groups = D / G;
    const uint32_t row_bytes = static_cast<uint32_t>(D * sizeof(T)), tile_bytes = TR * 2 * row_bytes;
    float* factors = reinterpret_cast<float*>(smem + static_cast<size_t>(stages) * tile_bytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t strip = blockIdx.x, vec = strip / p.strips_per_vec;
    const int64_t r_begin = vec * p.rows_per_vec + strip % p.strips_per_vec * p.strip_rows;
    const int rows = static_cast<int>(min(p.strip_rows, (vec + 1) * p.rows_per_vec - r_begin));
    const int tiles = (rows + TR - 1) / TR;
    const T* x = static_cast<const T*>(p.x) + r_begin * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + r_begin * p.ldy;
    // tile i (its rows of x, then those of dy) into stage s, by one warp: rows that
    // lie together in one copy (a copy per row: 165888 x 128 123 us, 65 so), else a
    // lane per row copy
    const bool whole_x = p.ldx == D, whole_dy = p.ldy == D;
    auto fill = [&](int i, int s) {
        const int n = min(TR, rows - i * TR);
        const int64_t r0 = int64_t(i) * TR;
        const uint32_t bar = smem_u32(full + s), to_x = smem_u32(smem) + s * tile_bytes, to_dy = to_x + TR * row_bytes;
        if (lane == 0) {
            mbar_arrive_expect_tx(bar, n * 2 * row_bytes);
            if (whole_x) bulk_load(to_x, x + r0 * p.ldx, n * row_bytes, bar);
            if (whole_dy) bulk_load(to_dy, dy + r0 * p.ldy, n * row_bytes, bar);
        }
        __syncwarp();
        if (!whole_x)
            for (int k = lane; k < n; k += 32) bulk_load(to_x + k * row_bytes, x + (r0 + k) * p.ldx, row_bytes, bar);
        if (!whole_dy)
            for (int k = lane; k < n; k += 32) bulk_load(to_dy + k * row_bytes, dy + (r0 + k) * p.ldy, row_bytes, bar);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(smem_u32(full + s), 1);
        abort_word = 0;
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    if (warp == 0)
        for (int i = 0; i < min(tiles, stages); ++i) fill(i, i);
    const V* w = p.weight ? static_cast<const V*>(p.weight) + vec * p.ldv : nullptr;
    // in planes of four elements per group, so that a warp's 16-byte reads hit distinct banks
    auto factor_at = [&](int c) { return c % G / 4 * (groups * 4) + c / G * 4 + c % 4; };
    for (int c = threadIdx.x; c < D; c += blockDim.x) factors[factor_at(c)] = w ? p.one + to_f(w[c]) : 1.0f;
    __syncthreads();

    // phase A: this warp's rows of a tile (a_row, a_row + NW / AP, ...) and its part of them
    constexpr int kStep = RL * CW / AP;
    const int a_row = warp / AP, a_part = warp % AP;
    float next_mean[AR], next_rstd[AR];
    auto prefetch = [&](int i) {
#pragma unroll
        for (int k = 0; k < AR; ++k) {
            const int r = i * TR + a_row + k * kStep;
            if (r < rows) {
                next_mean[k] = __ldg(p.mean + r_begin + r);
                next_rstd[k] = __ldg(p.rstd + r_begin + r);
            }
        }
    };
    prefetch(0);
    // phase B: this thread's columns and row lane
    const int row_lane = warp / CW, col_t = threadIdx.x - row_lane * 32 * CW;
    const Columns<T, kLay, 32 * CW> at{col_t, D};
    float2 fw[N][P], dw[N][P], db[N][P];
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < P; ++e) {
            fw[j][e] = at.some(j) ? *reinterpret_cast<const float2*>(factors + factor_at(at.column(j, 2 * e))) : both(0.0f);
            dw[j][e] = db[j][e] = both(0.0f);
        }
    T* dx = p.dx ? static_cast<T*>(p.dx) + (r_begin + row_lane) * p.D : nullptr;
    const float inv = 1.0f / static_cast<float>(D);
    int s = 0;
    uint32_t phase = 0;
    for (int i = 0; i < tiles; ++i) {
        const int flip = i & 1, n = min(TR, rows - i * TR);
        const uint8_t* tile = smem + static_cast<size_t>(s) * tile_bytes;
        mbar_wait(smem_u32(full + s), phase, &abort_word, Q6_SITE_NORM_RING);
        // ---------------------------------------------------------------- phase A
        float mean[AR], rstd[AR];
#pragma unroll
        for (int k = 0; k < AR; ++k) {
            mean[k] = next_mean[k];
            rstd[k] = next_rstd[k];
        }
        if (i + 1 < tiles) prefetch(i + 1);
#pragma unroll
        for (int k = 0; k < AR; ++k) {
            const int r = a_row + k * kStep;
            if (r < n) {
                const T* xr = reinterpret_cast<const T*>(tile + r * row_bytes);
                const T* yr = reinterpret_cast<const T*>(tile + (TR + r) * row_bytes);
                const float2 neg_mean = both(-mean[k]), scale = both(rstd[k]);
                float2 sa = both(0.0f), sh = both(0.0f);
#pragma unroll
                for (int j = 0; j < N * CW / AP; ++j) {
                    const int g = (j * AP + a_part) * 32 + lane;
                    if (kLay == kFull || g < groups) {
                        float2 fx[P], fy[P];
                        unpack(load_shared<T, G>(xr + g * G), fx);
                        unpack(load_shared<T, G>(yr + g * G), fy);
#pragma unroll
                        for (int e = 0; e < P; e += 2) {
                            const float4 f = *reinterpret_cast<const float4*>(factors + e / 2 * (groups * 4) + g * 4);
                            const float2 a0 = mul2(fy[e], make_float2(f.x, f.y)),
                                         a1 = mul2(fy[e + 1], make_float2(f.z, f.w));
                            sa = add2(sa, a0);
                            sh = fma2(a0, mul2(add2(fx[e], neg_mean), scale), sh);
                            sa = add2(sa, a1);
                            sh = fma2(a1, mul2(add2(fx[e + 1], neg_mean), scale), sh);
                        }
                    }
                }
                const float2 m = warp_sum2(make_float2(sa.x + sa.y, sh.x + sh.y));
                if (lane == 0) {
                    if constexpr (AP == 1) {
                        stats[flip][r] = make_float4(-mean[k], rstd[k], -m.x * inv, -m.y * inv);
                    } else {
                        parts[flip][r][a_part] = m;
                        if (a_part == 0) stats[flip][r] = make_float4(-mean[k], rstd[k], 0.0f, 0.0f);
                    }
                }
            }
        }
        __syncthreads();
        if (warp == 0 && i > 0 && i - 1 + stages < tiles) {  // tile i - 1 has been read by all
            fence_proxy_async_smem();
            fill(i - 1 + stages, s == 0 ? stages - 1 : s - 1);
        }
        // ---------------------------------------------------------------- phase B
#pragma unroll
        for (int q = 0; q < M; ++q) {
            const int r = row_lane + q * RL;
            if (r < n) {
                float4 row = stats[flip][r];
                if constexpr (AP > 1) {
                    float2 m = parts[flip][r][0];
                    if constexpr (AP % 2 == 0) {
                        const float4* pairs = reinterpret_cast<const float4*>(parts[flip][r]);
                        float4 two = pairs[0];
#pragma unroll
                        for (int k = 1; k < AP / 2; ++k) {
                            const float4 t = pairs[k];
                            two = make_float4(two.x + t.x, two.y + t.y, two.z + t.z, two.w + t.w);
                        }
                        m = make_float2(two.x + two.z, two.y + two.w);
                    } else {
#pragma unroll
                        for (int k = 1; k < AP; ++k) m = add2(m, parts[flip][r][k]);
                    }
                    row.z = -m.x * inv;
                    row.w = -m.y * inv;
                }
                const float2 neg_mean = both(row.x), rstd = both(row.y), kc = both(row.z), kh = both(row.w);
                const T* xr = reinterpret_cast<const T*>(tile + r * row_bytes);
                const T* yr = reinterpret_cast<const T*>(tile + (TR + r) * row_bytes);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    if (at.some(j)) {
                        float2 fx[P], fy[P];
                        unpack(load_shared<T, G>(xr + at.column(j, 0)), fx);
                        unpack(load_shared<T, G>(yr + at.column(j, 0)), fy);
#pragma unroll
                        for (int e = 0; e < P; ++e) {
                            const float2 h = mul2(add2(fx[e], neg_mean), rstd);
                            db[j][e] = add2(db[j][e], fy[e]);
                            dw[j][e] = fma2(fy[e], h, dw[j][e]);
                            fx[e] = mul2(fma2(fy[e], fw[j][e], fma2(h, kh, kc)), rstd);
                        }
                        if (dx) at.store(dx + (static_cast<int64_t>(i) * TR + q * RL) * p.D, j, pack<T, G>(fx));
                    }
                }
            }
        }
        if (++s == stages) {
            s = 0;
            phase ^= 1u;
        }
    }
    if (abort_word && threadIdx.x == 0)  // after a wait that gave up, no copy may outlive the CTA
        for (int i = max(0, tiles - stages); i < tiles; ++i)
            mbar_wait_drain(smem_u32(full + i % stages), static_cast<uint32_t>(i / stages & 1));
    if (!p.dw_part && !dweight && !p.db_part && !dbias) return;
    finish_columns<RL, 32 * CW>(p, at, row_lane, strip, reinterpret_cast<float*>(smem), dw, db, dweight, dbias);
}

// Backward of rows without 16-byte accesses: RL thread groups of CW warps, a row
// each, held in registers.
template <typename T, typename V, int CW, int N>
__global__ void __launch_bounds__(32 * CW * (CW < 16 ? 16 / CW : 1), 1)
    norm_grad_strided_kernel(const NormParams p, V* dweight, V* dbias) {
    constexpr int G = 16 / sizeof(T), P = G / 2, RL = CW < 16 ? 16 / CW : 1, kThreads = 32 * CW;
    static_assert(RL < 16 || CW == 1, "named barriers");
    __shared__ __align__(16) float2 parts[2][RL][CW];
    extern __shared__ __align__(128) uint8_t smem[];  // the column sums (finish_bytes)
    pdl_launch_dependents();
    pdl_wait();
    const int group = threadIdx.x / kThreads;
    const Columns<T, kStrided, kThreads> at{static_cast<int>(threadIdx.x) % kThreads, static_cast<int>(p.D)};
    const int64_t strip = blockIdx.x, vec = strip / p.strips_per_vec;
    const int64_t r_begin = vec * p.rows_per_vec + strip % p.strips_per_vec * p.strip_rows;
    const int64_t r_end = min(r_begin + p.strip_rows, (vec + 1) * p.rows_per_vec);
    const V* w = p.weight ? static_cast<const V*>(p.weight) + vec * p.ldv : nullptr;
    const float inv = 1.0f / static_cast<float>(at.D);
    float2 dw[N][P], db[N][P];
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) dw[j][i] = db[j][i] = both(0.0f);
    int flip = 0;
    for (int64_t r = r_begin + group; r < r_end; r += RL, flip ^= 1) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx;
        const T* dy = static_cast<const T*>(p.dy) + r * p.ldy;
        const float mean = __ldg(p.mean + r), rstd = __ldg(p.rstd + r);
        Group<T, G> gx[N], gy[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            gx[j] = at.load(x, j);
            gy[j] = at.load(dy, j);
        }
        float2 sa = both(0.0f), sh = both(0.0f);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (at.some(j)) {
                float2 fw[P], fx[P], fy[P];
                at.factor(w, j, p.one, fw);
                unpack(gx[j], fx);
                unpack(gy[j], fy);
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    const float2 h = mul2(add2(fx[e], both(-mean)), both(rstd)), a = mul2(fy[e], fw[e]);
                    dw[j][e] = fma2(fy[e], h, dw[j][e]);
                    db[j][e] = add2(db[j][e], fy[e]);
                    sa = add2(sa, a);
                    sh = fma2(a, h, sh);
                }
            }
        }
        if (!p.dx) continue;  // the same for the whole grid
        float2 m = warp_sum2(make_float2(sa.x + sa.y, sh.x + sh.y));
        if constexpr (CW > 1) {
            if ((at.t & 31) == 0) parts[flip][group][at.t >> 5] = m;
            asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kThreads) : "memory");
            m = parts[flip][group][0];
#pragma unroll
            for (int k = 1; k < CW; ++k) m = add2(m, parts[flip][group][k]);
        }
        const float2 ka = both(-m.x * inv), kh = both(-m.y * inv);
        // unpack the row again: in fp32 it would not fit the registers
#pragma unroll
        for (int j = 0; j < N; ++j) {
            keep_packed(gx[j]);
            keep_packed(gy[j]);
        }
        T* dx = static_cast<T*>(p.dx) + r * p.D;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (at.some(j)) {
                float2 fw[P], fx[P], fy[P];
                at.factor(w, j, p.one, fw);
                unpack(gx[j], fx);
                unpack(gy[j], fy);
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    const float2 h = mul2(add2(fx[e], both(-mean)), both(rstd));
                    fx[e] = mul2(fma2(fy[e], fw[e], fma2(h, kh, ka)), both(rstd));
                }
                at.store(dx, j, pack<T, G>(fx));
            }
        }
    }
    if (!p.dw_part && !dweight && !p.db_part && !dbias) return;
    finish_columns<RL, kThreads>(p, at, group, strip, reinterpret_cast<float*>(smem), dw, db, dweight, dbias);
}

}  // namespace norm_detail

// ------------------------------------------------------------------- host side

// W warps x N groups per thread cover a row (m: rows per thread and tile of the
// backward; lanes: of the warp, for one row); the first entry that covers the
// row's groups of G elements.
struct NormShape {
    int w, n, m = 1, lanes = 32;
};
constexpr NormShape kNormForward[] = {{1, 1, 1, 4}, {1, 1, 1, 8}, {1, 1, 1, 16}, {1, 1}, {1, 2},  {1, 4},  {2, 4},
                                      {3, 4},       {4, 4},       {6, 4},        {8, 4}, {12, 4}, {16, 4}, {32, 4}};
constexpr NormShape kNormGrad[] = {{1, 1, 4}, {1, 2, 2}, {2, 2, 2},  {3, 2, 3},  {4, 2, 2}, {6, 2, 2},
                                   {8, 2, 2}, {12, 2, 2}, {16, 2, 2}, {12, 4, 1}, {16, 4, 1}};
constexpr NormShape kNormGradStrided[] = {{1, 1, 1}, {1, 2, 1}, {2, 2, 1}, {4, 2, 1}, {8, 2, 1}, {16, 2, 1}, {16, 4, 1}};
constexpr int strided_row_lanes(int w) { return w < 16 ? 16 / w : 1; }

template <size_t K>
int norm_shape(const NormShape (&list)[K], int64_t D, int dtype) {
    const int64_t g = dtype == Q6_DTYPE_F32 ? 4 : 8, groups = (D + g - 1) / g;
    for (size_t i = 0; i < K; ++i)
        if (groups <= int64_t(list[i].lanes) * list[i].w * list[i].n) return static_cast<int>(i);
    return -1;  // the plain kernels
}

// Strips of rows for the column sums: about one per SM in all, each at least
// `least` rows (one per row lane).
void norm_plan_strips(int64_t M, int64_t rows_per_vec, int64_t least, int64_t* strip_rows, int64_t* strips_per_vec);

// Launches on one element type (a translation unit each); `vec` where every
// access can be 16 bytes, `shape` from the lists above.
template <typename T, typename V>
int norm_forward_typed(const NormParams& p, bool vec, int shape, cudaStream_t stream);
template <typename T, typename V>
int norm_grad_typed(const NormParams& p, bool vec, int shape, V* dweight, V* dbias, cudaStream_t stream);

template <typename T, typename V, norm_detail::Layout kLay, int W, int N, int L>
int launch_norm_forward(const NormParams& p, cudaStream_t stream) {
    auto* kernel = norm_detail::norm_kernel<T, V, kLay, W, N, L>;
    constexpr int threads = W == 1 ? 128 : 32 * W;
    // CTAs per SM, looked up once per device
    static std::atomic<int> resident[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return Q6_ERR_CUDA;
    if (dev < 0 || dev >= kMaxDevices) return Q6_ERR_UNSUPPORTED;
    int per_sm = resident[dev].load(std::memory_order_relaxed);
    if (per_sm == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0) != cudaSuccess || per_sm < 1)
            return Q6_ERR_CUDA;
        resident[dev].store(per_sm, std::memory_order_relaxed);
    }
    const int64_t rows = p.vecs ? p.rows_per_vec : p.M, vecs = p.vecs ? p.vecs : 1, per = W == 1 ? 128 / L : 1;
    const int64_t wave = std::max<int64_t>(1, int64_t(device_sm_count()) * per_sm / vecs);
    return launch_pdl(kernel, dim3(static_cast<unsigned>(std::min((rows + per - 1) / per, wave)), p.vecs ? p.vecs : 1u),
                      dim3(threads), 0, stream, p) == cudaSuccess
               ? Q6_OK
               : Q6_ERR_CUDA;
}

// Opts a kernel in to `bytes` of dynamic shared memory, once per device (a kernel
// has one caller, so the flags are the kernel's).
template <typename... A>
bool norm_opt_in(void (*kernel)(A...), int bytes, std::atomic<bool> (&done)[kMaxDevices]) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
    if (done[dev].load(std::memory_order_acquire)) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done[dev].store(true, std::memory_order_release);
    return true;
}

template <typename T, typename V, norm_detail::Layout kLay, int W, int N, int M>
int launch_norm_grad(const NormParams& p, V* dweight, V* dbias, cudaStream_t stream) {
    using namespace norm_detail;
    constexpr int lanes = grad_row_lanes(W), tile_rows = lanes * M;
    auto* kernel = norm_grad_kernel<T, V, kLay, W, N, M>;
    static std::atomic<bool> done[kMaxDevices];
    if (!norm_opt_in(kernel, kGradSmem, done)) return Q6_ERR_CUDA;
    const size_t factors = size_t(p.D) * sizeof(float), tile = size_t(tile_rows) * 2 * p.D * sizeof(T);
    const int64_t tiles = (std::min(p.strip_rows, p.rows_per_vec) + tile_rows - 1) / tile_rows;
    const int stages = static_cast<int>(
        std::min<int64_t>({int64_t(kGradMaxStages), tiles, static_cast<int64_t>((kGradSmem - factors) / tile)}));
    if (stages < std::min<int64_t>(2, tiles)) return Q6_ERR_UNSUPPORTED;  // a tile is refilled during the next one
    const size_t smem = std::max(stages * tile + factors, finish_bytes<lanes, 32 * W, N, 16 / int(sizeof(T))>());
    const int64_t strips = p.M / p.rows_per_vec * p.strips_per_vec;
    return launch_pdl(kernel, dim3(static_cast<unsigned>(strips)), dim3(32 * W * lanes), smem, stream, p, dweight,
                      dbias, stages) == cudaSuccess
               ? Q6_OK
               : Q6_ERR_CUDA;
}

template <typename T, typename V, int W, int N>
int launch_norm_grad_strided(const NormParams& p, V* dweight, V* dbias, cudaStream_t stream) {
    constexpr int lanes = strided_row_lanes(W);
    auto* kernel = norm_detail::norm_grad_strided_kernel<T, V, W, N>;
    constexpr size_t smem = norm_detail::finish_bytes<lanes, 32 * W, N, 16 / int(sizeof(T))>();
    static std::atomic<bool> done[kMaxDevices];
    if (!norm_opt_in(kernel, static_cast<int>(smem), done)) return Q6_ERR_CUDA;
    const int64_t strips = p.M / p.rows_per_vec * p.strips_per_vec;
    return launch_pdl(kernel, dim3(static_cast<unsigned>(strips)),
                      dim3(32 * W * lanes), smem, stream, p, dweight, dbias) == cudaSuccess
               ? Q6_OK
               : Q6_ERR_CUDA;
}

template <typename T, typename V, int W, int N, int L>
int norm_forward_layout(const NormParams& p, bool vec, cudaStream_t stream) {
    using namespace norm_detail;
    if (vec && p.D == L * W * N * int64_t(16 / sizeof(T))) return launch_norm_forward<T, V, kFull, W, N, L>(p, stream);
    return vec ? launch_norm_forward<T, V, kVec, W, N, L>(p, stream)
               : launch_norm_forward<T, V, kStrided, W, N, L>(p, stream);
}

template <typename T, typename V, int W, int N, int M>
int norm_grad_layout(const NormParams& p, V* dweight, V* dbias, cudaStream_t stream) {
    using namespace norm_detail;
    if (p.D == 32 * W * N * int64_t(16 / sizeof(T))) return launch_norm_grad<T, V, kFull, W, N, M>(p, dweight, dbias, stream);
    return launch_norm_grad<T, V, kVec, W, N, M>(p, dweight, dbias, stream);
}

template <typename T, typename V, size_t... I>
int norm_forward_list(const NormParams& p, bool vec, int shape, cudaStream_t stream, std::index_sequence<I...>) {
    int st = Q6_ERR_UNSUPPORTED;
    ((shape == int(I) &&
      (st = norm_forward_layout<T, V, kNormForward[I].w, kNormForward[I].n, kNormForward[I].lanes>(p, vec, stream), true)) ||
     ...);
    return st;
}

template <typename T, typename V, size_t... I>
int norm_grad_list(const NormParams& p, int shape, V* dweight, V* dbias, cudaStream_t stream, std::index_sequence<I...>) {
    int st = Q6_ERR_UNSUPPORTED;
    ((shape == int(I) &&
      (st = norm_grad_layout<T, V, kNormGrad[I].w, kNormGrad[I].n, kNormGrad[I].m>(p, dweight, dbias, stream), true)) ||
     ...);
    return st;
}

template <typename T, typename V, size_t... I>
int norm_grad_strided_list(const NormParams& p, int shape, V* dweight, V* dbias, cudaStream_t stream,
                           std::index_sequence<I...>) {
    int st = Q6_ERR_UNSUPPORTED;
    ((shape == int(I) && (st = launch_norm_grad_strided<T, V, kNormGradStrided[I].w, kNormGradStrided[I].n>(
                              p, dweight, dbias, stream),
                          true)) ||
     ...);
    return st;
}

// Device error words of the typed units.
int error_word_norm_bf16(bool clear);
int error_word_norm_f16(bool clear);
int error_word_norm_f32(bool clear);

#define Q6_NORM_UNIT(NAME)                                                                                        \
    int error_word_norm_##NAME(bool clear) {                                                                      \
        int v = 0;                                                                                                \
        if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return -1;                      \
        const int zero = 0;                                                                                       \
        if (clear && v != 0 && cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;  \
        return v;                                                                                                 \
    }

#define Q6_NORM_TYPES(T, V)                                                                                         \
    template <>                                                                                                     \
    int norm_forward_typed<T, V>(const NormParams& p, bool vec, int shape, cudaStream_t stream) {                   \
        return norm_forward_list<T, V>(p, vec, shape, stream, std::make_index_sequence<std::size(kNormForward)>{}); \
    }                                                                                                               \
    template <>                                                                                                     \
    int norm_grad_typed<T, V>(const NormParams& p, bool vec, int shape, V* dweight, V* dbias, cudaStream_t stream) { \
        return vec ? norm_grad_list<T, V>(p, shape, dweight, dbias, stream,                                         \
                                          std::make_index_sequence<std::size(kNormGrad)>{})                         \
                   : norm_grad_strided_list<T, V>(p, shape, dweight, dbias, stream,                                 \
                                                  std::make_index_sequence<std::size(kNormGradStrided)>{});         \
    }

}  // namespace q6
