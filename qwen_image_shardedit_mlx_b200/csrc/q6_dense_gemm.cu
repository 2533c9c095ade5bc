// Plans and launches the dense linear's products (q6_dense_gemm.cuh), and adds
// the partial sums of a split one.
#include "q6_dense_gemm.cuh"

#include <cudaTypedefs.h>

#include <cstdio>
#include <cstdlib>
#include <mutex>

namespace q6 {
namespace {

PFN_cuTensorMapEncodeTiled_v12000 dense_encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// Adds the split partials [splits][R][ldp] in split order and applies the
// epilogue; kVec: eight neighbouring outputs per thread.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) dense_reduce_kernel(const DenseParams p) {
    using namespace dense_detail;
    pdl_launch_dependents();
    pdl_wait();
    const int width = kVec ? p.C / 8 : p.C;
    const int64_t total = static_cast<int64_t>(p.R) * width;
    const int64_t plane = p.R * p.ld_partial;
    const DenseEpilogue& e = p.epi;
    for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int r = static_cast<int>(total >> 32 ? i / width : static_cast<uint32_t>(i) / static_cast<uint32_t>(width));
        const int c = static_cast<int>(i - int64_t(r) * width) * (kVec ? 8 : 1);
        const float* src = p.partial + r * p.ld_partial + c;
        const int gate_row = e.gate ? r / p.gate_rows : 0;
        if constexpr (kVec) {
            Eight<T> bias{}, gate{}, res{};
            if (e.bias) bias = load_ro<Eight<T>>(static_cast<const T*>(e.bias) + c);
            if (e.gate) gate = load_ro<Eight<T>>(gate_at<T>(e, gate_row, c));
            if (e.residual) res = *reinterpret_cast<const Eight<T>*>(static_cast<const T*>(e.residual) + r * e.ldr + c);
            float v[8] = {};
#pragma unroll 4
            for (int s = 0; s < p.splits; ++s) {
                const float4 a = *reinterpret_cast<const float4*>(src + s * plane);
                const float4 b = *reinterpret_cast<const float4*>(src + s * plane + 4);
                v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
                v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
            }
            finish8<T>(e, p.d, r, p.C, c, bias, gate, res, v);
        } else {
            T gate{}, res{};
            const float bias = e.bias ? to_f(load_ro<T>(static_cast<const T*>(e.bias) + c)) : 0.0f;
            if (e.gate) gate = load_ro<T>(gate_at<T>(e, gate_row, c));
            if (e.residual) res = static_cast<const T*>(e.residual)[r * e.ldr + c];
            float v = 0.0f;
#pragma unroll 4
            for (int s = 0; s < p.splits; ++s) v += src[s * plane];
            finish1<T>(e, p.d, int64_t(r) * p.C + c, bias, gate, res, v);
        }
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tile shape and split of one product: the least estimated time over the tile
// shapes.  In cycles: a stage costs the longer of its MMAs (2 CT per 64 of
// depth) and its operand bytes at 44 a cycle; a work item 700 more (ring fill,
// epilogue hand-over), a split the second kernel and its partials' traffic.  (A
// split joined within a cluster, each CTA's tile left in its shared memory, took
// as long: 9.5 us at 16 x 3072 -> 3072, 28 us at 256 x 12288 -> 3072.)
DensePlan plan_dense(int64_t R, int64_t C, int64_t L, bool q_t) {
    const int64_t sms = device_sm_count();
    struct Shape {
        int ct;
        bool pair;
    };
    static const Shape kShapes[] = {{256, true}, {192, true}, {128, true}, {128, false}, {64, false}, {32, false}, {16, false}};
    if (const char* v = std::getenv("Q6_DENSE_PLAN")) {  // "rows per tile,CTA pair,splits"
        int ct = 0, pair = 0, splits = 0;
        if (std::sscanf(v, "%d,%d,%d", &ct, &pair, &splits) == 3 && splits >= 1 && splits <= 16)
            for (const Shape& sh : kShapes)
                if (sh.ct == ct && sh.pair == (pair != 0) && !(q_t && (ct == 192 || ct < 64))) {
                    const int64_t stages = ceil_div(L, dense_stage_depth(ct)), per = ceil_div(stages, splits);
                    return DensePlan{ct, sh.pair, static_cast<int>(ceil_div(stages, per)), static_cast<int>(per)};
                }
    }
    DensePlan best{0, false, 1, 1};
    double best_cost = 0.0;
    for (const Shape& sh : kShapes) {
        if (q_t && (sh.ct == 192 || sh.ct < 64)) continue;
        const int depth = dense_stage_depth(sh.ct);
        const int64_t units = sh.pair ? sms / 2 : sms;
        const int64_t tiles = ceil_div(R, sh.ct) * ceil_div(C, sh.pair ? 256 : 128);
        const int64_t stages = ceil_div(L, depth);
        const double bytes = (128.0 + (sh.pair ? sh.ct / 2 : sh.ct)) * depth * 2;
        const double stage = std::max(2.0 * sh.ct * depth / 64, bytes / 44.0);
        const int64_t max_split = tiles >= units ? 1 : std::min<int64_t>({16, ceil_div(units, tiles), stages});
        for (int64_t s = 1; s <= max_split; ++s) {
            const int64_t per = ceil_div(stages, s);
            if (ceil_div(stages, per) != s) continue;
            const int64_t waves = ceil_div(tiles * s, units);
            double cost = waves * (per * stage + 700.0) + 2.0 * sh.ct;
            if (s > 1) cost += 5000.0 + s * (700.0 + R * C * 4 / 1500.0);
            if (best.ct == 0 || cost < best_cost) {
                best_cost = cost;
                best = DensePlan{sh.ct, sh.pair, static_cast<int>(s), static_cast<int>(per)};
            }
        }
    }
    return best;
}

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T>
int launch_reduce(const DenseParams& p, cudaStream_t stream) {
    const int64_t total = static_cast<int64_t>(p.R) * (p.vec ? p.C / 8 : p.C);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(ceil_div(total, 256), int64_t(device_sm_count()) * 8)));
    const cudaError_t e = p.vec ? launch_pdl(dense_reduce_kernel<T, true>, grid, dim3(256), 0, stream, p)
                                : launch_pdl(dense_reduce_kernel<T, false>, grid, dim3(256), 0, stream, p);
    return e == cudaSuccess ? Q6_OK : Q6_ERR_CUDA;
}

}  // namespace

bool dense_tensor_map(CUtensorMap* map, int dtype, const void* base, int64_t inner, int64_t outer, int64_t ld,
                      int box_outer) {
    auto fn = dense_encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    const cuuint32_t box[2] = {kDenseBox, static_cast<cuuint32_t>(box_outer)};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, dtype == Q6_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
              const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t dense_product_workspace_bytes(int64_t R, int64_t C, int64_t L, bool, bool q_t) {
    const DensePlan plan = plan_dense(R, C, L, q_t);
    return plan.splits > 1 ? static_cast<size_t>(plan.splits) * R * (ceil_div(C, 8) * 8) * sizeof(float) : 0;
}

int launch_dense_product(const DenseProduct& a, cudaStream_t stream) {
    const DensePlan plan = plan_dense(a.R, a.C, a.L, a.q_t);
    DenseParams p{};
    p.d = a.d;
    p.epi = a.epi;
    p.R = static_cast<int>(a.R);
    p.C = static_cast<int>(a.C);
    p.gate_rows = a.epi.gate ? static_cast<int>(a.epi.rows_per_gate) : p.R;
    const DenseEpilogue& e = a.epi;
    p.vec = a.C % 8 == 0 && al16(a.d) && al16(e.bias) && al16(e.gate) && al16(e.residual) && al16(e.preact) &&
            (!e.gate || e.ldg % 8 == 0) && (!e.residual || e.ldr % 8 == 0);
    p.half = a.dtype == Q6_DTYPE_F16;
    const int64_t tiles_r = ceil_div(a.R, plan.ct), tile_c = plan.pair ? 256 : 128, tiles_c = ceil_div(a.C, tile_c);
    if (tiles_r * tiles_c * plan.splits > (int64_t(1) << 30)) return Q6_ERR_UNSUPPORTED;
    p.tiles_r = static_cast<int>(tiles_r);
    p.tiles_c = static_cast<int>(tiles_c);
    p.splits = plan.splits;
    p.stages_per_split = plan.stages_per_split;
    p.k_stages = static_cast<int>(ceil_div(a.L, dense_stage_depth(plan.ct)));
    p.num_items = static_cast<int>(tiles_r * tiles_c * plan.splits);
    // rows walked together: one wave's tiles about square, in groups of equal height
    const int64_t units = device_sm_count() / (plan.pair ? 2 : 1);
    int64_t want = 1;
    while (want * want * plan.ct < units * tile_c) ++want;
    const int64_t groups = ceil_div(tiles_r, want);
    p.group_r = static_cast<int>(ceil_div(tiles_r, groups));
    p.ld_partial = ceil_div(a.C, 8) * 8;
    if (plan.splits > 1) {
        const size_t need = static_cast<size_t>(plan.splits) * a.R * p.ld_partial * sizeof(float);
        if (!a.workspace || a.workspace_bytes < need) return Q6_ERR_WORKSPACE;
        p.partial = static_cast<float*>(a.workspace);
    }
    const int st = !a.p_t   ? launch_dense_nn(a, p, plan, stream)
                   : !a.q_t ? launch_dense_tn(a, p, plan, stream)
                            : launch_dense_tt(a, p, plan, stream);
    if (st != Q6_OK || plan.splits == 1) return st;
    return p.half ? launch_reduce<__half>(p, stream) : launch_reduce<__nv_bfloat16>(p, stream);
}

int error_word_dense(bool clear) {
    int code = 0;
    for (const int w : {error_word_dense_nn(clear), error_word_dense_tn(clear), error_word_dense_tt(clear)}) {
        if (w < 0) return -1;
        if (code == 0) code = w;
    }
    return code;
}

}  // namespace q6
