// Dense linear for a few rows (1 to 16): bound by reading the weight once.
//
//   y[m, n] = epilogue(sum_k x[m, k] W[n, k])
//
// A CTA takes 16 rows of W; its warps share the sum, 128 of k at a time (64 from
// nine rows of x on, which are two MMA tiles).  The products run on warp-level
// MMAs (m16n8k16) with the weight rows as the A operand and the rows of x as B,
// straight from global memory: within a block of 32 of k
// lane t of a row holds eight neighbouring values (one 16-byte load), and since
// both operands number the sum's terms the same way, the MMA's own order of them
// does not matter.  So the weight passes through no shared memory and no
// shuffles; eight 16-byte loads of it per lane are in flight per turn.  The warps'
// partial sums meet in shared memory and are added in order.
//
// bf16, one row: 3072 -> 18432 19.5 us (5.8 TB/s), 3072 -> 3072 6.3 us, 12288 -> 3072
// 15.1 us; the tcgen05 path, which needs a second kernel for its split sums, takes
// 20.9, 9.2 and 17.8.  (dense_few_rows has the figures of sixteen rows.)
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "q6_dense.cuh"
#include "q6_dense.h"
#include "q6_internal.h"
#include "q6_ptx.cuh"

namespace q6 {
namespace {

constexpr int kTileN = 16;     // weight rows per CTA
// Blocks of 32 of k per turn (unaligned rows load two groups for each value's
// group), and warps per CTA at most: two such CTAs fit an SM's registers, 64 a
// thread.
template <bool kAligned, int MT>
constexpr int kBlocks = (kAligned ? 4 : 2) / MT;
constexpr int kMaxWarps = 16;
constexpr int kTileM = 8;  // rows of x per MMA; MT such tiles

struct RowsParams {
    const void* x;
    const void* w;
    void* y;
    int64_t ldx, ldw;
    int M, N, K;
    int gate_rows;
    DenseEpilogue epi;
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight values of a row from k on, zero past K, by element (any alignment).
__device__ __forceinline__ uint4 load8_each(const uint16_t* row, int k, int K) {
    uint4 v;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = k + 2 * i < K ? __ldg(row + k + 2 * i) : 0u;
        const uint32_t hi = k + 2 * i + 1 < K ? __ldg(row + k + 2 * i + 1) : 0u;
        w[i] = lo | hi << 16;
    }
    return v;
}

// The two aligned 16-byte groups around eight values of any alignment, and the
// values shifted out of them.
struct Around {
    uint4 a, b;
};
__device__ __forceinline__ Around load_around(const uint16_t* at) {
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(at) & ~uintptr_t(15));
    return {__ldg(p), __ldg(p + 1)};
}
__device__ __forceinline__ uint4 shift_out(const Around& g, uint32_t off) {
    uint32_t w0 = g.a.x, w1 = g.a.y, w2 = g.a.z, w3 = g.a.w, w4 = g.b.x, w5 = g.b.y;
    if (off & 8) w0 = g.a.z, w1 = g.a.w, w2 = g.b.x, w3 = g.b.y, w4 = g.b.z, w5 = g.b.w;
    if (off & 4) w0 = w1, w1 = w2, w2 = w3, w3 = w4, w4 = w5;
    const uint32_t bits = (off & 2) * 8;
    return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                      __funnelshift_r(w3, w4, bits));
}

// One turn's eight-value groups of a row, k0 + 32 i + 8 t on.  Rows that are not
// aligned 16-byte groups: where `inner` says that the groups around all of them
// lie inside the operand (and before K), two aligned loads and a shift each; else
// by element, which is for the ends of a sum (by element throughout, 6 x 9985 ->
// 8729 took 93 us, 46 so).
template <bool kAligned, int B>
__device__ __forceinline__ void load_turn(const uint16_t* row, int k, int K, bool inner, uint4 (&v)[B]) {
    if constexpr (kAligned) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (k + 32 * i < K) v[i] = __ldg(reinterpret_cast<const uint4*>(row + k + 32 * i));
        }
    } else if (inner) {
        Around g[B];
#pragma unroll
        for (int i = 0; i < B; ++i) g[i] = load_around(row + k + 32 * i);
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + k)) & 15;
#pragma unroll
        for (int i = 0; i < B; ++i) v[i] = shift_out(g[i], off);
    } else {
#pragma unroll
        for (int i = 0; i < B; ++i) v[i] = load8_each(row, k + 32 * i, K);
    }
}

template <typename T, bool kAligned, int MT>
__global__ void __launch_bounds__(kMaxWarps * 32, 2) dense_rows_kernel(const RowsParams p) {
    constexpr int B = kBlocks<kAligned, MT>, kTurn = 32 * B;
    __shared__ float sums[kMaxWarps][MT * kTileM][kTileN + 1];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * kTileN;
    // rows beyond the weight read its last one and are not stored; rows beyond x are zeros
    const uint16_t* w0 = static_cast<const uint16_t*>(p.w) + int64_t(min(n0 + g, p.N - 1)) * p.ldw;
    const uint16_t* w1 = static_cast<const uint16_t*>(p.w) + int64_t(min(n0 + g + 8, p.N - 1)) * p.ldw;
    const uint16_t* x = static_cast<const uint16_t*>(p.x) + g * p.ldx;
    pdl_wait();
    float c[MT][4] = {};
    for (int k0 = warp * kTurn; k0 < p.K; k0 += warps * kTurn) {
        uint4 a0[B], a1[B], b[MT][B];
        // the groups around a turn's values reach at most eight values beyond it
        const bool before = k0 + kTurn + 8 <= p.K;
        const bool inner = before && (k0 >= 8 || n0 > 0);
        load_turn<kAligned>(w0, k0 + 8 * t, p.K, inner, a0);
        load_turn<kAligned>(w1, k0 + 8 * t, p.K, inner, a1);
#pragma unroll
        for (int h = 0; h < MT; ++h) {
            if (g + h * kTileM < p.M) {
                load_turn<kAligned>(x + h * kTileM * p.ldx, k0 + 8 * t, p.K, before && k0 >= 8, b[h]);
            } else {
#pragma unroll
                for (int i = 0; i < B; ++i) b[h][i] = make_uint4(0u, 0u, 0u, 0u);
            }
        }
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int h = 0; h < MT; ++h) {
                mma16816<T>(c[h], a0[i].x, a1[i].x, a0[i].y, a1[i].y, b[h][i].x, b[h][i].y);
                mma16816<T>(c[h], a0[i].z, a1[i].z, a0[i].w, a1[i].w, b[h][i].z, b[h][i].w);
            }
    }
    // c: weight rows g and g + 8, rows 2 t and 2 t + 1 of a tile of x
#pragma unroll
    for (int h = 0; h < MT; ++h) {
        float(*to)[kTileN + 1] = sums[warp] + h * kTileM + 2 * t;
        to[0][g] = c[h][0];
        to[1][g] = c[h][1];
        to[0][g + 8] = c[h][2];
        to[1][g + 8] = c[h][3];
    }
    __syncthreads();
    const DenseEpilogue& e = p.epi;
    for (int i = threadIdx.x; i < p.M * kTileN; i += blockDim.x) {
        const int m = i / kTileN, n = n0 + i % kTileN;
        if (n >= p.N) continue;
        float v = 0.0f;
        for (int k = 0; k < warps; ++k) v += sums[k][m][i % kTileN];
        if (e.bias) v = __fadd_rn(v, to_f(static_cast<const T*>(e.bias)[n]));
        const int64_t at = int64_t(m) * p.N + n;
        if (e.preact) {
            if (e.preact_f32)
                static_cast<float*>(e.preact)[at] = v;
            else
                static_cast<__half*>(e.preact)[at] = preact_half(v);
        }
        v = act_f(v, e.activation);
        if (e.gate) v = __fmul_rn(v, to_f(static_cast<const T*>(e.gate)[m / p.gate_rows * e.ldg + n]));
        if (e.residual) v = __fadd_rn(v, to_f(static_cast<const T*>(e.residual)[m * e.ldr + n]));
        static_cast<T*>(p.y)[at] = from_f<T>(v);
    }
}

template <typename T, bool kAligned, int MT>
cudaError_t launch_tiles(const RowsParams& p, cudaStream_t stream) {
    constexpr int kTurn = 32 * kBlocks<kAligned, MT>;
    // as many warps as let every CTA run at once, no more than the turns of one sum
    const int64_t tiles = (p.N + kTileN - 1) / kTileN, turns = (p.K + kTurn - 1) / kTurn;
    const int64_t per_sm = (tiles + device_sm_count() - 1) / device_sm_count();
    const int64_t warps = std::max<int64_t>(
        1, std::min<int64_t>({2 * kMaxWarps / per_sm, turns, int64_t(kMaxWarps)}));
    return launch_pdl(dense_rows_kernel<T, kAligned, MT>, dim3(static_cast<unsigned>(tiles)),
                      dim3(static_cast<unsigned>(32 * warps)), 0, stream, p);
}

template <typename T, bool kAligned>
cudaError_t launch_typed(const RowsParams& p, cudaStream_t stream) {
    return p.M <= kTileM ? launch_tiles<T, kAligned, 1>(p, stream) : launch_tiles<T, kAligned, 2>(p, stream);
}

}  // namespace

// Here against the tcgen05 path, bf16, in us.
// Up to eight rows: one row 1024 -> 1024 2.9 / 6.6, 3072 -> 64 3.4 / 7.2, 12288 -> 64
// 7.4 / 9.1, 12288 -> 3072 15.2 / 19.0, 3072 -> 18432 20.0 / 21.5; eight rows 3.1 / 6.7,
// 3.5 / 7.2, 7.5 / 9.4, 16.9 / 19.7, 21.1 / 21.8; nearest 12288 -> 1024, 11.3 / 11.8 and
// 12.6 / 12.1.  The sum is not split over CTAs, so a longer one with few outputs
// takes longer here: one row 18432 -> 128 12.7 / 11.2, 49152 -> 64 27.7 / 15.6.  The rule
// has no case for those: no layer here sums over more than 12288.
// To sixteen, x is as large as a CTA's part of the weight, and an SM takes in both:
// the tcgen05 path, which reads x once per 128 rows of W, wins where the sum is long
// or the weight large: 768 -> 768 2.8 / 5.7, 3072 -> 3072 7.9 / 9.5, 4096 -> 4096
// 10.0 / 12.1, 6144 -> 3072 12.6 / 13.5, 3072 -> 9216 13.3 / 15.3; 3072 -> 12288
// 17.7 / 17.1, 9216 -> 3072 17.5 / 16.4, 12288 -> 1024 17.5 / 11.8.
bool dense_few_rows(int64_t R, int64_t C, int64_t L) {
    return R <= kTileM || (R <= 2 * kTileM && L <= 6144 && C * L <= (int64_t(1) << 25));
}

int launch_dense_rows(const DenseProduct& a, cudaStream_t stream) {
    RowsParams p{};
    p.x = a.q;
    p.w = a.p;
    p.y = a.d;
    p.ldx = a.ldq;
    p.ldw = a.ldp;
    p.M = static_cast<int>(a.R);
    p.N = static_cast<int>(a.C);
    p.K = static_cast<int>(a.L);
    p.gate_rows = a.epi.gate ? static_cast<int>(a.epi.rows_per_gate) : p.M;
    p.epi = a.epi;
    const bool aligned = p.K % 8 == 0 && p.ldw % 8 == 0 && p.ldx % 8 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0 &&
                         reinterpret_cast<uintptr_t>(p.x) % 16 == 0;
    cudaError_t e;
    if (a.dtype == Q6_DTYPE_F16)
        e = aligned ? launch_typed<__half, true>(p, stream) : launch_typed<__half, false>(p, stream);
    else
        e = aligned ? launch_typed<__nv_bfloat16, true>(p, stream) : launch_typed<__nv_bfloat16, false>(p, stream);
    return e == cudaSuccess ? Q6_OK : Q6_ERR_CUDA;
}

}  // namespace q6
