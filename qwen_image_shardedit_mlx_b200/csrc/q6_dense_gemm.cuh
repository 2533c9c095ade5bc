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
// allow that (odd widths, odd addresses) take one output per lane instead.
//
// Every mbarrier wait is bounded (q6_ptx.cuh).
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

// Epilogue of eight neighbouring outputs of row r starting at column c.
template <typename T>
__device__ __forceinline__ void finish8(const DenseEpilogue& e, void* d, int64_t r, int64_t C, int c, int64_t gate_row,
                                        const Eight<T>& bias, const Eight<T>& residual, float (&v)[8]) {
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fadd_rn(v[i], to_f(bias.v[i]));
    }
    const int64_t at = r * C + c;
    if (e.preact) {
        if (e.preact_f32) {
            float4* z = reinterpret_cast<float4*>(static_cast<float*>(e.preact) + at);
            z[0] = make_float4(v[0], v[1], v[2], v[3]);
            z[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            Eight<__half> z;
#pragma unroll
            for (int i = 0; i < 8; ++i) z.v[i] = preact_half(v[i]);
            *reinterpret_cast<Eight<__half>*>(static_cast<__half*>(e.preact) + at) = z;
        }
    }
    if (e.activation == Q6_ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_f(v[i], Q6_ACT_GELU_TANH);
    } else if (e.activation == Q6_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_f(v[i], Q6_ACT_SILU);
    }
    if (e.gate) {
        const Eight<T> g = *reinterpret_cast<const Eight<T>*>(static_cast<const T*>(e.gate) + gate_row * e.ldg + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], to_f(g.v[i]));
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

// The same for kRows outputs of one column c (rows r .. r + n - 1 of them), any
// layout; the rows' loads are issued together.  kPlain: a bias at most.
template <typename T, int kRows, bool kPlain>
__device__ __forceinline__ void finish_column(const DenseEpilogue& e, void* d, int r, int n, int64_t C, int c,
                                              int gate_rows, float bias, float (&v)[kRows]) {
    T* y = static_cast<T*>(d) + r * C + c;
    if constexpr (kPlain) {
#pragma unroll
        for (int i = 0; i < kRows; ++i, y += C)
            if (i < n) *y = from_f<T>(__fadd_rn(v[i], bias));
    } else {
        T res[kRows], gate[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (i < n) {
                if (e.residual) res[i] = static_cast<const T*>(e.residual)[(r + i) * e.ldr + c];
                if (e.gate) gate[i] = static_cast<const T*>(e.gate)[(r + i) / gate_rows * e.ldg + c];
            }
        }
        int64_t at = r * C + c;
#pragma unroll
        for (int i = 0; i < kRows; ++i, at += C, y += C) {
            if (i < n) {
                float t = __fadd_rn(v[i], bias);
                if (e.preact) {
                    if (e.preact_f32)
                        static_cast<float*>(e.preact)[at] = t;
                    else
                        static_cast<__half*>(e.preact)[at] = preact_half(t);
                }
                t = act_f(t, e.activation);
                if (e.gate) t = __fmul_rn(t, to_f(gate[i]));
                if (e.residual) t = __fadd_rn(t, to_f(res[i]));
                *y = from_f<T>(t);
            }
        }
    }
}

// One warp's 32 columns (lanes of tensor memory) x kChunk rows.
template <typename T, int kChunk>
__device__ __forceinline__ void dense_epilogue_block(const DenseParams& p, const DenseItem& I, uint32_t taddr,
                                                     float* stage, int r0, int c0, const Eight<T>& bias) {
    const int lane = threadIdx.x & 31;
    const DenseEpilogue& e = p.epi;
    const int cv = c0 + (lane & 3) * 8;
    Eight<T> res[kChunk / 8];
    const bool to_partial = p.splits > 1;
    if (p.vec && !to_partial && e.residual) {  // in flight while the accumulator is read
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {
            const int r = r0 + i * 8 + (lane >> 2);
            if (r < p.R && cv < p.C)
                res[i] = *reinterpret_cast<const Eight<T>*>(static_cast<const T*>(e.residual) + r * e.ldr + cv);
        }
    }
    uint32_t v[kChunk];
    if constexpr (kChunk == 32)
        tmem_ld_32x32b_x32(taddr, v);
    else
        tmem_ld_32x32b_x16(taddr, v);
    tmem_wait_ld();
    // stage[row][column], the 16-byte groups of odd rows swapped in pairs so that
    // the reads below (two rows, every other group) hit distinct banks
#pragma unroll
    for (int j = 0; j < kChunk; ++j) stage[j * 32 + (lane ^ ((j & 1) << 2))] = __uint_as_float(v[j]);
    __syncwarp();
    if (p.vec || to_partial) {
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {
            const int j = i * 8 + (lane >> 2), g = (lane & 3) * 2, odd = j & 1;
            const float4 a = *reinterpret_cast<const float4*>(stage + j * 32 + ((g ^ odd) << 2));
            const float4 b = *reinterpret_cast<const float4*>(stage + j * 32 + (((g + 1) ^ odd) << 2));
            float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            const int r = r0 + j;
            if (r < p.R && cv < p.C) {
                if (to_partial) {
                    float4* dst = reinterpret_cast<float4*>(
                        p.partial + (static_cast<int64_t>(I.split) * p.R + r) * p.ld_partial + cv);
                    dst[0] = a;
                    dst[1] = b;
                } else {
                    finish8<T>(e, p.d, r, p.C, cv, e.gate ? r / p.gate_rows : 0, bias, res[i], f);
                }
            }
        }
    } else {
        const int c = c0 + lane;
        if (c < p.C) {
            const float b = e.bias ? to_f(static_cast<const T*>(e.bias)[c]) : 0.0f;
            const bool plain = !e.preact && e.activation == Q6_ACT_NONE && !e.gate && !e.residual;
#pragma unroll 1
            for (int j = 0; j < kChunk && r0 + j < p.R; j += 8) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = stage[(j + i) * 32 + (lane ^ ((i & 1) << 2))];
                const int n = min(8, p.R - r0 - j);
                if (plain && n == 8)
                    finish_column<T, 8, true>(e, p.d, r0 + j, 8, p.C, c, p.gate_rows, b, f);
                else
                    finish_column<T, 8, false>(e, p.d, r0 + j, n, p.C, c, p.gate_rows, b, f);
            }
        }
    }
    __syncwarp();
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
                    dense_epilogue_block<__half, C::kChunk>(p, I, taddr + ch * C::kChunk, stage, r0, c0,
                                                            *reinterpret_cast<const Eight<__half>*>(&bias));
                else
                    dense_epilogue_block<__nv_bfloat16, C::kChunk>(p, I, taddr + ch * C::kChunk, stage, r0, c0,
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
