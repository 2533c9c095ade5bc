// Matrix product of the dense linear on the tensor cores:
//
//   d[r, c] = epilogue(sum_l Q(r, l) P(c, l))      16-bit operands, fp32 sums
//
// The MMA computes the transpose: its 128 lanes (256 for a CTA pair) are
// columns c of d and its N side is a tile of CT rows r, so one orientation
// serves a single row (CT = 16) and thousands (CT = 256), and the lanes of a
// warp always hold neighbouring outputs of a row.  Each operand is stored with
// l contiguous (K-major) or transposed (its index contiguous, MN-major): TMA
// boxes of 64 elements of the contiguous axis with 128-byte swizzling either
// way, and the tcgen05 shared-memory descriptors read both orders.  So the
// forward product (x, W), the input's gradient (dz, W^T) and the weight's
// gradient (dz^T, x^T) are the same kernel without a transposed copy.
//
// Warp 0 feeds a ring of TMA stages, warp 1 issues the MMAs, warps 4-11 run
// the epilogue of one accumulator while the MMAs fill the other (two per SM in
// tensor memory).  The CTA (pair) is persistent over tiles; tiles are walked in
// groups of rows so that one wave's operands stay in L2.  Where the tiles leave
// SMs idle the sum is split: fp32 partial tiles, added in split order by
// dense_reduce_kernel, which then applies the epilogue.
//
// The epilogue moves 32 x 32 blocks through shared memory (fp32, per warp), so
// that each lane ends up with eight neighbouring outputs of a row: 16-byte
// loads of bias, gate and residual and 16-byte stores.  Layouts that do not
// allow that (odd widths, odd addresses) take one column per lane instead.
//
// Every mbarrier wait is bounded (q6_ptx.cuh) and begins after the previous kernel's
// end, so that its limit covers this kernel's own pipeline alone.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "q6_dense.cuh"
#include "q6_dense.h"
#include "q6_internal.h"
#include "q6_ptx.cuh"

namespace q6 {

struct DenseParams {
    void* d;
    DenseEpilogue epi;
    int R, C;
    int gate_rows;       // rows per gate vector
    bool vec;            // 16-byte epilogue accesses are possible
    bool half;           // fp16 (else bf16)
    int tiles_r, tiles_c, num_items;
    int group_r;         // row tiles walked together
    int k_stages, splits, stages_per_split;
    float* partial;      // [splits, R, ldp] when splits > 1
    int64_t ld_partial;  // C rounded up to 8
};

// What one launch runs (chosen by plan_dense).
struct DensePlan {
    int ct;  // rows of d per tile
    bool pair;
    int splits, stages_per_split;
};

constexpr int kDenseLanes = 128;  // columns of d per CTA
constexpr int kDenseBox = 64;     // elements along the contiguous axis per TMA box
constexpr int kDenseEpiWarps = 8;
constexpr int kDenseThreads = 128 + 32 * kDenseEpiWarps;
constexpr int kDenseSmem = 227 * 1024;
constexpr int kDenseStaging = kDenseEpiWarps * 32 * 32 * 4;

// Depth of the sum per pipeline stage: 64, or 128 for the narrow tiles, whose
// MMAs are too short to hide a barrier round trip per 64.
__host__ __device__ constexpr int dense_stage_depth(int ct) { return ct >= 128 ? 64 : 128; }

template <int CT, bool kPair, bool kQT>
struct DenseCfg {
    static constexpr int kBoxes = dense_stage_depth(CT) / kDenseBox;
    static constexpr int kQRows = kPair ? CT / 2 : CT;             // rows of Q this CTA stages
    static constexpr int kPBytes = kDenseLanes * kDenseBox * 2;    // per 64 of depth
    static constexpr int kQBytes = kQRows * kDenseBox * 2;
    static constexpr int kStageBytes = kBoxes * (kPBytes + kQBytes);
    static constexpr int kStages = (kDenseSmem - 1024 - 512 - kDenseStaging) / kStageBytes;
    static constexpr int kSmemBytes = 1024 + 512 + kDenseStaging + kStages * kStageBytes;
    static constexpr int kTmemCols = CT <= 16 ? 32 : CT <= 32 ? 64 : CT <= 64 ? 128 : CT <= 128 ? 256 : 512;
    static constexpr int kChunk = CT < 32 ? CT : 32;               // rows per epilogue block
    static_assert(CT % 16 == 0 && CT >= 16 && CT <= 256, "MMA N");
    static_assert(!kQT || kQRows % kDenseBox == 0, "transposed Q is staged in boxes of 64 rows");
    static_assert(kStages >= 3 && kStages <= 16, "stage ring");
    static_assert(kQBytes % 1024 == 0, "swizzle atoms");
};

namespace dense_detail {

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void mma_ss_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Descriptor high half: 128-byte swizzle, sm_100 version, stride 1024 (eight
// 128-byte rows); low half: start address and, for MN-major tiles, the leading
// stride between 64-element chunks of the index (a 64 x 64 box: 8192 bytes).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);

template <bool kT>
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem) {
    return ((smem & 0x3FFFFu) >> 4) | ((kT ? (8192u >> 4) : 1u) << 16);
}

// Start-address step (16-byte units) per MMA depth of 16: 32 bytes along a
// K-major row, sixteen 128-byte rows of an MN-major box.
template <bool kT>
constexpr uint32_t kStep16 = kT ? (16 * 128) >> 4 : 32 >> 4;

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int site) {
    // lane 0 decides for the warp, so a timeout is seen by all lanes alike
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, abort_flag, site) ? 1 : 0;
    ok = __shfl_sync(0xffffffffu, ok, 0);
    if (ok) (void)mbar_try_wait(bar, parity);  // every lane observes the completed phase itself
    return ok != 0;
}

struct DenseItem {
    int r, c, split, s0, s1;
};

__device__ __forceinline__ DenseItem dense_item(const DenseParams& p, int it) {
    DenseItem I;
    I.split = it % p.splits;
    int tile = it / p.splits;
    const int per_group = p.group_r * p.tiles_c;
    const int g = tile / per_group;
    tile -= g * per_group;
    const int rows = min(p.group_r, p.tiles_r - g * p.group_r);
    I.c = tile / rows;
    I.r = g * p.group_r + tile % rows;
    I.s0 = I.split * p.stages_per_split;
    I.s1 = min(I.s0 + p.stages_per_split, p.k_stages);
    return I;
}

template <typename T>
struct alignas(16) Eight {
    T v[8];
};

// z of kCols neighbouring outputs, for the backward pass.
template <int kCols>
__device__ __forceinline__ void store_preact(const DenseEpilogue& e, int64_t at, const float* v) {
    if (e.preact_f32) {
        float* z = static_cast<float*>(e.preact) + at;
        if constexpr (kCols == 8) {
            reinterpret_cast<float4*>(z)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(z)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *z = v[0];
        }
    } else {
        __half* z = static_cast<__half*>(e.preact) + at;
        if constexpr (kCols == 8) {
            Eight<__half> g;
#pragma unroll
            for (int i = 0; i < 8; ++i) g.v[i] = preact_half(v[i]);
            *reinterpret_cast<Eight<__half>*>(z) = g;
        } else {
            *z = preact_half(v[0]);
        }
    }
}

// A warp's block through shared memory, stage[row][column]: the 16-byte groups of
// odd rows are swapped in pairs, so that the reads (two rows, every other group)
// hit distinct banks.
template <int kChunk>
__device__ __forceinline__ void stage_block(float* stage, const uint32_t (&v)[kChunk]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < kChunk; ++j) stage[j * 32 + (lane ^ ((j & 1) << 2))] = __uint_as_float(v[j]);
    __syncwarp();
}
// Row j's eight columns from 8 (lane % 4) on.
__device__ __forceinline__ void read_stage(const float* stage, int j, float* f) {
    const int g = (threadIdx.x & 3) * 2, odd = j & 1;
    const float4 a = *reinterpret_cast<const float4*>(stage + j * 32 + ((g ^ odd) << 2));
    const float4 b = *reinterpret_cast<const float4*>(stage + j * 32 + (((g + 1) ^ odd) << 2));
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
    f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// Epilogue of eight neighbouring outputs of row r starting at column c.
template <typename T>
__device__ __forceinline__ void finish8(const DenseEpilogue& e, void* d, int64_t r, int64_t C, int c,
                                        const Eight<T>& bias, const Eight<T>& gate, const Eight<T>& residual,
                                        float (&v)[8]) {
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fadd_rn(v[i], to_f(bias.v[i]));
    }
    const int64_t at = r * C + c;
    if (e.preact) store_preact<8>(e, at, v);
    if (e.activation == Q6_ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_f(v[i], Q6_ACT_GELU_TANH);
    } else if (e.activation == Q6_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_f(v[i], Q6_ACT_SILU);
    }
    if (e.gate) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], to_f(gate.v[i]));
    }
    if (e.residual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fadd_rn(v[i], to_f(residual.v[i]));
    }
    Eight<T> y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] = from_f<T>(v[i]);
    *reinterpret_cast<Eight<T>*>(static_cast<T*>(d) + at) = y;
}

// The same for one output.
template <typename T>
__device__ __forceinline__ void finish1(const DenseEpilogue& e, void* d, int64_t at, float bias, T gate, T residual,
                                        float v) {
    v = __fadd_rn(v, bias);
    if (e.preact) store_preact<1>(e, at, &v);
    v = act_f(v, e.activation);
    if (e.gate) v = __fmul_rn(v, to_f(gate));
    if (e.residual) v = __fadd_rn(v, to_f(residual));
    static_cast<T*>(d)[at] = from_f<T>(v);
}

template <typename T>
__device__ __forceinline__ const T* gate_at(const DenseEpilogue& e, int64_t gate_row, int c) {
    return static_cast<const T*>(e.gate) + gate_row * e.ldg + c;
}

// What one warp's block of the epilogue covers: 32 columns (lanes of tensor memory)
// x kChunk rows.  By eight a lane has rows lane / 4, + 8, ... and eight columns from
// c on, else every row and column c.
struct DenseBlock {
    int r0, rows, c;
    bool inside, one_gate;  // c is a column of d; the rows share a gate vector
    int gate_row;           // of the first row
};

template <int kChunk>
__device__ __forceinline__ void load_accumulator(uint32_t taddr, uint32_t (&v)[kChunk]) {
    __syncwarp();  // lanes outside the columns may have skipped loads
    if constexpr (kChunk == 32)
        tmem_ld_32x32b_x32(taddr, v);
    else
        tmem_ld_32x32b_x16(taddr, v);
    tmem_wait_ld();
}

// A bias at most.  kAllRows: the block has all of its rows.
template <typename T, int kChunk, bool kAllRows>
__device__ __forceinline__ void dense_epilogue_plain(const DenseParams& p, const DenseBlock& B, uint32_t taddr,
                                                     float* stage, const Eight<T>& bias8) {
    const int lane = threadIdx.x & 31;
    const DenseEpilogue& e = p.epi;
    const float bias = !p.vec && e.bias && B.inside ? to_f(load_ro<T>(static_cast<const T*>(e.bias) + B.c)) : 0.0f;
    uint32_t v[kChunk];
    load_accumulator<kChunk>(taddr, v);
    T* y = static_cast<T*>(p.d) + B.r0 * int64_t(p.C) + B.c;
    if (p.vec) {
        stage_block<kChunk>(stage, v);
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {
            const int j = i * 8 + (lane >> 2);
            float f[8];
            read_stage(stage, j, f);
            Eight<T> out;
#pragma unroll
            for (int k = 0; k < 8; ++k) out.v[k] = from_f<T>(e.bias ? __fadd_rn(f[k], to_f(bias8.v[k])) : f[k]);
            if ((kAllRows || j < B.rows) && B.inside) *reinterpret_cast<Eight<T>*>(y + j * int64_t(p.C)) = out;
        }
        __syncwarp();
    } else if (B.inside) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i, y += p.C)
            if (kAllRows || i < B.rows) *y = from_f<T>(e.bias ? __fadd_rn(__uint_as_float(v[i]), bias) : __uint_as_float(v[i]));
    }
}

// A block with all of its rows, one gate vector at most: straight passes over
// sixteen of the lane's values, without a condition per row, so that their
// latencies overlap (an SM has eight epilogue warps).  What the passes read is
// loaded one turn ahead; the residual so before the rows of y, which may lie in it,
// are written.  In turns of sixteen because a short sum runs the epilogue once per
// CTA, and its time is then that of fetching its instructions: with all 32 values
// in one turn 580 x 240 -> 2696 (GELU, gate, residual) took 14.4 us, 11.3 so;
// 8192 x 1001 -> 777 (gate, residual), which the latencies bound, 51 and 46, and 118
// with loops over the rows.
template <typename T, int kChunk, bool kEight>
__device__ __forceinline__ void dense_epilogue_full(const DenseParams& p, const DenseBlock& B, uint32_t taddr, float* stage,
                                                    const Eight<T>& bias8) {
    constexpr int kPart = 16, kRows = kEight ? kPart / 8 : kPart, kCols = kEight ? 8 : 1;
    const int lane = threadIdx.x & 31;
    const DenseEpilogue& e = p.epi;
    const int first = B.r0 + (kEight ? lane >> 2 : 0), step = kEight ? 8 : 1;
    const T* from = static_cast<const T*>(e.residual) + first * e.ldr + B.c;
    Eight<T> gate{}, next[2];
    float bias = 0.0f;
    auto load_residual = [&] {
#pragma unroll
        for (int i = 0; i < kRows; ++i, from += step * e.ldr) {
            if constexpr (kEight)
                next[i] = *reinterpret_cast<const Eight<T>*>(from);
            else
                next[i / 8].v[i % 8] = *from;
        }
    };
    if (B.inside) {
        if (e.residual) load_residual();
        if (e.gate) {
            if constexpr (kEight)
                gate = load_ro<Eight<T>>(gate_at<T>(e, B.gate_row, B.c));
            else
                gate.v[0] = load_ro<T>(gate_at<T>(e, B.gate_row, B.c));
        }
        if (!kEight && e.bias) bias = to_f(load_ro<T>(static_cast<const T*>(e.bias) + B.c));
    }
    uint32_t v[kChunk];
    load_accumulator<kChunk>(taddr, v);
    const int64_t row = step * int64_t(p.C);
    int64_t at = first * int64_t(p.C) + B.c;
    stage_block<kChunk>(stage, v);
    if (B.inside) {
#pragma unroll 1
        for (int h = 0; h < kChunk / kPart; ++h) {
            const Eight<T> res[2] = {next[0], next[1]};
            if (e.residual && h + 1 < kChunk / kPart) load_residual();
            float f[kPart];
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                if constexpr (kEight)
                    read_stage(stage, h * kPart + i * 8 + (lane >> 2), f + 8 * i);
                else
                    f[i] = stage[(h * kPart + i) * 32 + (lane ^ ((i & 1) << 2))];
            }
            if (e.bias) {
#pragma unroll
                for (int i = 0; i < kPart; ++i) f[i] = __fadd_rn(f[i], kEight ? to_f(bias8.v[i % 8]) : bias);
            }
            if (e.preact) {
#pragma unroll
                for (int i = 0; i < kRows; ++i) store_preact<kCols>(e, at + i * row, f + kCols * i);
            }
            if (e.activation == Q6_ACT_GELU_TANH) {
#pragma unroll
                for (int i = 0; i < kPart; ++i) f[i] = act_f(f[i], Q6_ACT_GELU_TANH);
            } else if (e.activation == Q6_ACT_SILU) {
#pragma unroll
                for (int i = 0; i < kPart; ++i) f[i] = act_f(f[i], Q6_ACT_SILU);
            }
            if (e.gate) {
#pragma unroll
                for (int i = 0; i < kPart; ++i) f[i] = __fmul_rn(f[i], to_f(gate.v[kEight ? i % 8 : 0]));
            }
            if (e.residual) {
#pragma unroll
                for (int i = 0; i < kPart; ++i) f[i] = __fadd_rn(f[i], to_f(res[i / 8].v[i % 8]));
            }
            T* y = static_cast<T*>(p.d) + at;
#pragma unroll
            for (int i = 0; i < kRows; ++i, y += row) {
                if constexpr (kEight) {
                    Eight<T> out;
#pragma unroll
                    for (int k = 0; k < 8; ++k) out.v[k] = from_f<T>(f[8 * i + k]);
                    *reinterpret_cast<Eight<T>*>(y) = out;
                } else {
                    *y = from_f<T>(f[i]);
                }
            }
            at += kRows * row;
        }
    }
    __syncwarp();
}

// Any block of outputs, by eight or one.
template <typename T, int kChunk>
__device__ __forceinline__ void dense_epilogue_ragged(const DenseParams& p, const DenseBlock& B, uint32_t taddr,
                                                      float* stage, const Eight<T>& bias8) {
    const int lane = threadIdx.x & 31;
    const DenseEpilogue& e = p.epi;
    uint32_t v[kChunk];
    load_accumulator<kChunk>(taddr, v);
    stage_block<kChunk>(stage, v);
    if (B.inside) {
        if (p.vec) {
#pragma unroll 1
            for (int j = lane >> 2; j < B.rows; j += 8) {
                const int r = B.r0 + j;
                Eight<T> gate{}, res{};
                if (e.gate) gate = load_ro<Eight<T>>(gate_at<T>(e, r / p.gate_rows, B.c));
                if (e.residual)
                    res = *reinterpret_cast<const Eight<T>*>(static_cast<const T*>(e.residual) + r * e.ldr + B.c);
                float f[8];
                read_stage(stage, j, f);
                finish8<T>(e, p.d, r, p.C, B.c, bias8, gate, res, f);
            }
        } else {
            const float bias = e.bias ? to_f(load_ro<T>(static_cast<const T*>(e.bias) + B.c)) : 0.0f;
#pragma unroll 1
            for (int j = 0; j < B.rows; j += 4) {
                T gate[4], res[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = B.r0 + j + i;
                    if (j + i < B.rows) {
                        if (e.gate) gate[i] = load_ro<T>(gate_at<T>(e, r / p.gate_rows, B.c));
                        if (e.residual) res[i] = static_cast<const T*>(e.residual)[r * e.ldr + B.c];
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (j + i < B.rows)
                        finish1<T>(e, p.d, (B.r0 + j + i) * int64_t(p.C) + B.c, bias, gate[i], res[i],
                                   stage[(j + i) * 32 + (lane ^ ((i & 1) << 2))]);
            }
        }
    }
    __syncwarp();
}

// kPlain: a product with no epilogue (the gradients').
template <typename T, int kChunk, bool kPlain>
__device__ __forceinline__ void dense_epilogue_block(const DenseParams& p, const DenseItem& I, uint32_t taddr,
                                                     float* stage, int r0, int c0, const Eight<T>& bias) {
    const int lane = threadIdx.x & 31;
    DenseBlock B;
    B.r0 = r0;
    B.rows = min(kChunk, p.R - r0);
    if (p.splits > 1) {
        float* to = p.partial + (static_cast<int64_t>(I.split) * p.R + r0) * p.ld_partial;
        const int c = c0 + (lane & 3) * 8;
        uint32_t v[kChunk];
        load_accumulator<kChunk>(taddr, v);
        stage_block<kChunk>(stage, v);
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {  // by eight: a partial row is padded to that
            const int j = i * 8 + (lane >> 2);
            if (j < B.rows && c < p.C) {
                float f[8];
                read_stage(stage, j, f);
                float4* dst = reinterpret_cast<float4*>(to + j * p.ld_partial + c);
                dst[0] = make_float4(f[0], f[1], f[2], f[3]);
                dst[1] = make_float4(f[4], f[5], f[6], f[7]);
            }
        }
        __syncwarp();
        return;
    }
    B.c = c0 + (p.vec ? (lane & 3) * 8 : lane);
    B.inside = B.c < p.C;
    const bool all_rows = B.rows == kChunk;
    if constexpr (kPlain) {
        if (all_rows)
            dense_epilogue_plain<T, kChunk, true>(p, B, taddr, stage, bias);
        else
            dense_epilogue_plain<T, kChunk, false>(p, B, taddr, stage, bias);
    } else {
        const DenseEpilogue& e = p.epi;
        B.gate_row = 0;
        B.one_gate = true;
        if (e.gate) {
            B.gate_row = r0 / p.gate_rows;
            B.one_gate = (r0 + B.rows - 1) / p.gate_rows == B.gate_row;
        }
        if (!all_rows || !B.one_gate)
            dense_epilogue_ragged<T, kChunk>(p, B, taddr, stage, bias);
        else if (!e.preact && e.activation == Q6_ACT_NONE && !e.gate && !e.residual)
            dense_epilogue_plain<T, kChunk, true>(p, B, taddr, stage, bias);
        else if (p.vec)
            dense_epilogue_full<T, kChunk, true>(p, B, taddr, stage, bias);
        else
            dense_epilogue_full<T, kChunk, false>(p, B, taddr, stage, bias);
    }
}

template <int CT, bool kPair, bool kPT, bool kQT>
__global__ void __launch_bounds__(kDenseThreads, 1)
    dense_product_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
                         const DenseParams p) {
    using C = DenseCfg<CT, kPair, kQT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_align_up<1024>(smem_raw);
    float* staging = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStageBytes + kDenseStaging);
    uint64_t* full = bars;
    uint64_t* empty = bars + 16;
    uint64_t* acc_full = bars + 32;
    uint64_t* acc_empty = bars + 34;
    uint64_t* drain = bars + 36;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 37);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 38);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = kPair ? cluster_ctarank() : 0u;
    const bool leader = rank == 0;
    const int it0 = kPair ? blockIdx.x >> 1 : blockIdx.x, istep = kPair ? gridDim.x >> 1 : gridDim.x;
    constexpr int kTileC = kPair ? 2 * kDenseLanes : kDenseLanes;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(smem_u32(full + i), 1);
            mbar_init(smem_u32(empty + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(acc_full + i), 1);
            mbar_init(smem_u32(acc_empty + i), kDenseEpiWarps * (kPair ? 2 : 1));
        }
        mbar_init(smem_u32(drain), 1);
        fence_mbar_init();
    }
    if (warp == 2) {
        if constexpr (kPair) {
            tmem_alloc_pair(smem_u32(tmem_slot), C::kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kPair) cluster_sync();  // the peer's barriers are initialised
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            tma_prefetch_map(&tmap_p);
            tma_prefetch_map(&tmap_q);
            pdl_wait();
            uint32_t s = 0, ph = 0;
            long issued = 0;
            bool ok = true;
            for (int it = it0; it < p.num_items && ok; it += istep) {
                const DenseItem I = dense_item(p, it);
                const int c0 = I.c * kTileC + static_cast<int>(rank) * kDenseLanes;
                const int r0 = I.r * CT + static_cast<int>(rank) * C::kQRows * (kPair ? 1 : 0);
                for (int ks = I.s0; ks < I.s1; ++ks) {
                    if (!mbar_wait(smem_u32(empty + s), ph ^ 1u, abort_flag, 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = smem_u32(full + s);
                    const uint32_t fbc = kPair ? mapa_shared(fb, 0) : fb;
                    if (leader) mbar_arrive_expect_tx(fb, (kPair ? 2u : 1u) * C::kStageBytes);
                    const uint32_t dst = smem_u32(smem + s * C::kStageBytes);
                    auto load = [&](uint32_t to, const CUtensorMap* map, int x, int y) {
                        if constexpr (kPair)
                            tma_load_2d_pair(to, map, fbc, x, y);
                        else
                            tma_load_2d(to, map, fbc, x, y);
                    };
#pragma unroll
                    for (int b = 0; b < C::kBoxes; ++b) {
                        const int l = (ks * C::kBoxes + b) * kDenseBox;
                        const uint32_t pd = dst + b * C::kPBytes;
                        const uint32_t qd = dst + C::kBoxes * C::kPBytes + b * C::kQBytes;
                        if constexpr (kPT) {
                            load(pd, &tmap_p, c0, l);
                            load(pd + 8192, &tmap_p, c0 + kDenseBox, l);
                        } else {
                            load(pd, &tmap_p, l, c0);
                        }
                        if constexpr (kQT) {
#pragma unroll
                            for (int h = 0; h < C::kQRows / kDenseBox; ++h)
                                load(qd + h * 8192, &tmap_q, r0 + h * kDenseBox, l);
                        } else {
                            load(qd, &tmap_q, l, r0);
                        }
                    }
                    ++issued;
                    if (++s == C::kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            // every copy lands, and every MMA that reads it retires, before this CTA may exit
            const long tail = issued < C::kStages ? issued : C::kStages;
            for (long i = 0; i < tail; ++i) {
                const long n = issued - 1 - i;
                mbar_wait_drain(smem_u32(empty + n % C::kStages), static_cast<uint32_t>((n / C::kStages) & 1));
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        // The whole warp walks the loop so that the operands stay warp-uniform;
        // one elected lane issues a stage's MMAs and their commit.
        if (leader) {
            // before the first timed wait: the previous kernel may run for longer than its limit
            pdl_wait();
            const uint32_t idesc = (1u << 4) | ((p.half ? 0u : 1u) << 7) | ((p.half ? 0u : 1u) << 10) |
                                   ((kPT ? 1u : 0u) << 15) | ((kQT ? 1u : 0u) << 16) |
                                   (static_cast<uint32_t>(CT >> 3) << 17) | (static_cast<uint32_t>(kTileC >> 4) << 24);
            const uint32_t p_lo = desc_lo<kPT>(smem_u32(smem));
            const uint32_t q_lo = desc_lo<kQT>(smem_u32(smem) + C::kBoxes * C::kPBytes);
            uint32_t s = 0, ph = 0, acc = 0, accph = 0;
            bool ok = true;
            for (int it = it0; it < p.num_items && ok; it += istep) {
                const DenseItem I = dense_item(p, it);
                if (!warp_wait(smem_u32(acc_empty + acc), accph ^ 1u, abort_flag, 2)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * CT;
                for (int ks = I.s0; ks < I.s1; ++ks) {
                    if (!warp_wait(smem_u32(full + s), ph, abort_flag, 3)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t off = s * (C::kStageBytes >> 4);
                    const uint32_t first = ks != I.s0 ? 1u : 0u;
                    if (elect_one()) {
#pragma unroll
                        for (int b = 0; b < C::kBoxes; ++b)
#pragma unroll
                            for (int kk = 0; kk < kDenseBox / 16; ++kk) {
                                const uint64_t pd =
                                    make_desc(p_lo + off + b * (C::kPBytes >> 4) + kk * kStep16<kPT>, kDescHi);
                                const uint64_t qd =
                                    make_desc(q_lo + off + b * (C::kQBytes >> 4) + kk * kStep16<kQT>, kDescHi);
                                if constexpr (kPair)
                                    mma_ss_pair(d_tmem, pd, qd, idesc, b + kk == 0 ? first : 1u);
                                else
                                    mma_ss(d_tmem, pd, qd, idesc, b + kk == 0 ? first : 1u);
                            }
                        if constexpr (kPair)
                            tc_commit_pair(smem_u32(empty + s), 3);
                        else
                            tc_commit(smem_u32(empty + s));
                    }
                    __syncwarp();
                    if (++s == C::kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (!ok) break;
                if (elect_one()) {
                    if constexpr (kPair)
                        tc_commit_pair(smem_u32(acc_full + acc), 3);
                    else
                        tc_commit(smem_u32(acc_full + acc));
                }
                __syncwarp();
                if (++acc == 2) {
                    acc = 0;
                    accph ^= 1u;
                }
            }
            // all issued MMAs complete before tensor memory is released
            if (elect_one()) {
                if constexpr (kPair)
                    tc_commit_pair(smem_u32(drain), 1);
                else
                    tc_commit(smem_u32(drain));
                mbar_wait_drain(smem_u32(drain), 0);
            }
            __syncwarp();
        }
    } else if (warp >= 4) {
        // ------------------------------------------------ epilogue
        const int ew = warp - 4, quarter = warp & 3, half_cols = ew >> 2;
        float* stage = staging + ew * 1024;
        pdl_wait();  // d, the residual, the gate and the partials may be the previous kernel's
        uint32_t acc = 0, accph = 0;
        for (int it = it0; it < p.num_items; it += istep) {
            const DenseItem I = dense_item(p, it);
            const int c0 = I.c * kTileC + static_cast<int>(rank) * kDenseLanes + quarter * 32;
            const int cv = c0 + (lane & 3) * 8;
            uint4 bias = make_uint4(0u, 0u, 0u, 0u);
            if (p.vec && p.splits == 1 && p.epi.bias && cv < p.C)
                bias = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.epi.bias) + cv);
            if (!warp_wait(smem_u32(acc_full + acc), accph, abort_flag, 4)) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * CT;
#pragma unroll 1
            for (int ch = half_cols; ch < CT / C::kChunk; ch += 2) {
                const int r0 = I.r * CT + ch * C::kChunk;
                if (r0 >= p.R) break;  // the same for the whole warp
                if (p.half)
                    dense_epilogue_block<__half, C::kChunk, kPT>(p, I, taddr + ch * C::kChunk, stage, r0, c0,
                                                                 *reinterpret_cast<const Eight<__half>*>(&bias));
                else
                    dense_epilogue_block<__nv_bfloat16, C::kChunk, kPT>(
                        p, I, taddr + ch * C::kChunk, stage, r0, c0,
                        *reinterpret_cast<const Eight<__nv_bfloat16>*>(&bias));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (kPair)
                    mbar_arrive_cluster(mapa_shared(smem_u32(acc_empty + acc), 0));
                else
                    mbar_arrive(smem_u32(acc_empty + acc));
            }
            if (++acc == 2) {
                acc = 0;
                accph ^= 1u;
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if constexpr (kPair) cluster_sync();  // the leader's MMAs into this CTA's tensor memory have retired
    if (warp == 2) {
        tc_fence_after();
        if constexpr (kPair)
            tmem_dealloc_pair(tmem_base, C::kTmemCols);
        else
            tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

}  // namespace dense_detail

// ------------------------------------------------------------------- host side

bool dense_tensor_map(CUtensorMap* map, int dtype, const void* base, int64_t inner, int64_t outer, int64_t ld,
                      int box_outer);

template <int CT, bool kPair, bool kPT, bool kQT>
int launch_dense_tile(const DenseProduct& a, DenseParams p, cudaStream_t stream) {
    using C = DenseCfg<CT, kPair, kQT>;
    auto* kernel = dense_detail::dense_product_kernel<CT, kPair, kPT, kQT>;
    static std::atomic<bool> attr_set_for_device[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return Q6_ERR_CUDA;
    if (dev < 0 || dev >= kMaxDevices) return Q6_ERR_UNSUPPORTED;
    if (!attr_set_for_device[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes) != cudaSuccess)
            return Q6_ERR_CUDA;
        attr_set_for_device[dev].store(true, std::memory_order_release);
    }
    CUtensorMap mp, mq;
    const bool ok = (kPT ? dense_tensor_map(&mp, a.dtype, a.p, a.C, a.L, a.ldp, kDenseBox)
                         : dense_tensor_map(&mp, a.dtype, a.p, a.L, a.C, a.ldp, kDenseLanes)) &&
                    (kQT ? dense_tensor_map(&mq, a.dtype, a.q, a.R, a.L, a.ldq, kDenseBox)
                         : dense_tensor_map(&mq, a.dtype, a.q, a.L, a.R, a.ldq, C::kQRows));
    if (!ok) return Q6_ERR_CUDA;
    const int units = device_sm_count() / (kPair ? 2 : 1);
    const int workers = std::min(p.num_items, units);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(workers * (kPair ? 2 : 1)));
    cfg.blockDim = dim3(kDenseThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (kPair) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 2;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = static_cast<unsigned>(n);
    return cudaLaunchKernelEx(&cfg, kernel, mp, mq, static_cast<const DenseParams>(p)) == cudaSuccess ? Q6_OK
                                                                                                     : Q6_ERR_CUDA;
}

// One tile shape per call, by operand order (one translation unit each).
int launch_dense_nn(const DenseProduct& a, const DenseParams& p, const DensePlan& plan, cudaStream_t stream);
int launch_dense_tn(const DenseProduct& a, const DenseParams& p, const DensePlan& plan, cudaStream_t stream);
int launch_dense_tt(const DenseProduct& a, const DenseParams& p, const DensePlan& plan, cudaStream_t stream);

// Device error words of those units (as the error_word_* functions of q6_internal.h).
int error_word_dense_nn(bool clear);
int error_word_dense_tn(bool clear);
int error_word_dense_tt(bool clear);

template <bool kPT, bool kQT>
int launch_dense_order(const DenseProduct& a, const DenseParams& p, const DensePlan& plan, cudaStream_t stream) {
    if (plan.pair) {
        switch (plan.ct) {
            case 256: return launch_dense_tile<256, true, kPT, kQT>(a, p, stream);
            case 192:
                if constexpr (!kQT) return launch_dense_tile<192, true, kPT, kQT>(a, p, stream);
                break;
            case 128: return launch_dense_tile<128, true, kPT, kQT>(a, p, stream);
        }
        return Q6_ERR_UNSUPPORTED;
    }
    switch (plan.ct) {
        case 128: return launch_dense_tile<128, false, kPT, kQT>(a, p, stream);
        case 64: return launch_dense_tile<64, false, kPT, kQT>(a, p, stream);
        case 32:
            if constexpr (!kQT) return launch_dense_tile<32, false, kPT, kQT>(a, p, stream);
            break;
        case 16:
            if constexpr (!kQT) return launch_dense_tile<16, false, kPT, kQT>(a, p, stream);
            break;
    }
    return Q6_ERR_UNSUPPORTED;
}

#define Q6_DENSE_UNIT(NAME, PT, QT)                                                                                  \
    int launch_dense_##NAME(const DenseProduct& a, const DenseParams& p, const DensePlan& plan, cudaStream_t stream) { \
        return launch_dense_order<PT, QT>(a, p, plan, stream);                                                       \
    }                                                                                                                \
    int error_word_dense_##NAME(bool clear) {                                                                        \
        int v = 0;                                                                                                   \
        if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return -1;                         \
        const int zero = 0;                                                                                          \
        if (clear && v != 0 && cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;     \
        return v;                                                                                                    \
    }

}  // namespace q6
