// Layer norm over rows of D, forward and gradients (q6_layer_norm,
// q6_layer_norm_grad):
//   y = xh w + b,  xh = (x - mean) rstd
//   a = dy w,  dx = rstd (a - mean_D(a) - xh mean_D(a xh)),
//   dweight = sum over rows of dy xh,  dbias = sum over rows of dy.
// Statistics and sums in fp32 (the variance from centred values, a second
// pass); one rounding at each output.
#include <algorithm>
#include <cstdint>

#include "q6_dense.cuh"
#include "q6_internal.h"
#include "q6_ptx.cuh"

namespace q6 {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;

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
};

__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[kThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) t += part[i];
    return t;
}

// One CTA per row, any width, stride and alignment.
template <typename T, typename V>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(NormParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < p.D; i += kThreads) s += to_f(x[i]);
    const float mean = block_sum(s) / static_cast<float>(p.D);
    float q = 0.0f;
    for (int64_t i = threadIdx.x; i < p.D; i += kThreads) {
        const float c = to_f(x[i]) - mean;
        q = fmaf(c, c, q);
    }
    const float rstd = rsqrtf(block_sum(q) / static_cast<float>(p.D) + p.eps);
    if (p.mean && threadIdx.x == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    const int64_t v0 = row / p.rows_per_vec * p.ldv;
    const V* w = static_cast<const V*>(p.weight);
    const V* b = static_cast<const V*>(p.bias);
    T* y = static_cast<T*>(p.y) + row * p.D;
    for (int64_t i = threadIdx.x; i < p.D; i += kThreads) {
        const float f = w ? p.one + to_f(w[v0 + i]) : 1.0f;
        y[i] = from_f<T>(fmaf((to_f(x[i]) - mean) * rstd, f, b ? to_f(b[v0 + i]) : 0.0f));
    }
}

template <typename T, typename V>
__global__ void __launch_bounds__(kThreads) norm_rows_dx_kernel(NormParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + row * p.ldy;
    const V* w = p.weight ? static_cast<const V*>(p.weight) + row / p.rows_per_vec * p.ldv : nullptr;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s = 0.0f, q = 0.0f;
    for (int64_t i = threadIdx.x; i < p.D; i += kThreads) {
        const float a = to_f(dy[i]) * (w ? p.one + to_f(w[i]) : 1.0f);
        s += a;
        q = fmaf(a, (to_f(x[i]) - mean) * rstd, q);
    }
    s = block_sum(s) / static_cast<float>(p.D);
    q = block_sum(q) / static_cast<float>(p.D);
    T* dx = static_cast<T*>(p.dx) + row * p.D;
    for (int64_t i = threadIdx.x; i < p.D; i += kThreads) {
        const float a = to_f(dy[i]) * (w ? p.one + to_f(w[i]) : 1.0f);
        dx[i] = from_f<T>(rstd * (a - s - (to_f(x[i]) - mean) * rstd * q));
    }
}

// Partial column sums of dy xh and dy over one strip of rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_column_sums_kernel(NormParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t strip = blockIdx.x / p.col_blocks;
    const int64_t c = blockIdx.x % p.col_blocks * int64_t(kThreads) + threadIdx.x;
    if (c >= p.D) return;
    const int64_t v = strip / p.strips_per_vec;
    const int64_t r0 = v * p.rows_per_vec + strip % p.strips_per_vec * p.strip_rows;
    const int64_t r1 = std::min(r0 + p.strip_rows, (v + 1) * p.rows_per_vec);
    float dw = 0.0f, db = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float g = to_f(static_cast<const T*>(p.dy)[r * p.ldy + c]);
        db += g;
        dw = fmaf(g, (to_f(static_cast<const T*>(p.x)[r * p.ldx + c]) - p.mean[r]) * p.rstd[r], dw);
    }
    if (p.dw_part) p.dw_part[strip * p.D + c] = dw;
    if (p.db_part) p.db_part[strip * p.D + c] = db;
}

template <typename V>
__global__ void __launch_bounds__(128) norm_sum_strips_kernel(const float* __restrict__ part, int64_t strips_per_vec,
                                                              int64_t D, V* out) {
    pdl_launch_dependents();
    pdl_wait();
    const unsigned col_blocks = static_cast<unsigned>((D + 127) / 128);
    const int64_t c = blockIdx.x % col_blocks * int64_t(128) + threadIdx.x, v = blockIdx.x / col_blocks;
    if (c >= D) return;
    float t = 0.0f;
#pragma unroll 8
    for (int64_t i = 0; i < strips_per_vec; ++i) t += part[(v * strips_per_vec + i) * D + c];
    out[v * D + c] = from_f<V>(t);
}

void plan_strips(int64_t M, int64_t rows_per_vec, int64_t* strip_rows, int64_t* strips_per_vec) {
    const int64_t vecs = M / rows_per_vec, want = std::max<int64_t>(1, 592 / vecs);
    *strip_rows = std::max<int64_t>(1, (rows_per_vec + want - 1) / want);
    *strips_per_vec = (rows_per_vec + *strip_rows - 1) / *strip_rows;
}

size_t round_up(size_t v) { return (v + 255) / 256 * 256; }

size_t grad_bytes(int64_t M, int64_t D, int64_t rows_per_vec, int outputs) {
    int64_t rows, per;
    plan_strips(M, rows_per_vec, &rows, &per);
    const size_t part = round_up(size_t(M / rows_per_vec) * per * D * sizeof(float));
    return ((outputs & Q6_GRAD_W) ? part : 0) + ((outputs & Q6_GRAD_BIAS) ? part : 0);
}

template <typename T, typename V>
int run_forward(const NormParams& p, cudaStream_t stream) {
    return launch_pdl(norm_rows_kernel<T, V>, dim3(static_cast<unsigned>(p.M)), dim3(kThreads), 0, stream, p) ==
                   cudaSuccess
               ? Q6_OK
               : Q6_ERR_CUDA;
}

template <typename T, typename V>
int run_grad(const NormParams& p, void* dweight, void* dbias, cudaStream_t stream) {
    if (p.dx && launch_pdl(norm_rows_dx_kernel<T, V>, dim3(static_cast<unsigned>(p.M)), dim3(kThreads), 0, stream,
                           p) != cudaSuccess)
        return Q6_ERR_CUDA;
    if (!dweight && !dbias) return Q6_OK;
    const int64_t vecs = p.M / p.rows_per_vec, strips = vecs * p.strips_per_vec, sum_blocks = (p.D + 127) / 128;
    if (strips * p.col_blocks > kMaxGrid || vecs * sum_blocks > kMaxGrid) return Q6_ERR_UNSUPPORTED;
    if (launch_pdl(norm_column_sums_kernel<T>, dim3(static_cast<unsigned>(strips * p.col_blocks)), dim3(kThreads), 0,
                   stream, p) != cudaSuccess)
        return Q6_ERR_CUDA;
    const dim3 grid(static_cast<unsigned>(vecs * sum_blocks));
    if (dweight && launch_pdl(norm_sum_strips_kernel<V>, grid, dim3(128), 0, stream,
                              static_cast<const float*>(p.dw_part), p.strips_per_vec, p.D,
                              static_cast<V*>(dweight)) != cudaSuccess)
        return Q6_ERR_CUDA;
    if (dbias && launch_pdl(norm_sum_strips_kernel<V>, grid, dim3(128), 0, stream,
                            static_cast<const float*>(p.db_part), p.strips_per_vec, p.D,
                            static_cast<V*>(dbias)) != cudaSuccess)
        return Q6_ERR_CUDA;
    return Q6_OK;
}

// Calls f with the element types of dtype / vec_dtype.
template <typename F>
int with_types(int dtype, int vec_dtype, F&& f) {
    const bool wide = vec_dtype == Q6_DTYPE_F32;
    if (dtype == Q6_DTYPE_F32) return f(float{}, float{});
    if (dtype == Q6_DTYPE_F16) return wide ? f(__half{}, float{}) : f(__half{}, __half{});
    return wide ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

int check_norm(const void* x, int64_t ldx, int64_t ldv, int64_t rows_per_vec, int64_t M, int64_t D, int dtype,
               int vec_dtype, int flags, bool has_vec) {
    if (!x || M <= 0 || D <= 0 || M > kMaxGrid || D > (int64_t(1) << 30)) return Q6_ERR_INVALID_ARGUMENT;
    if (dtype < Q6_DTYPE_BF16 || dtype > Q6_DTYPE_F32) return Q6_ERR_UNSUPPORTED;
    if (vec_dtype != dtype && vec_dtype != Q6_DTYPE_F32) return Q6_ERR_UNSUPPORTED;
    if (rows_per_vec <= 0 || rows_per_vec > M || M % rows_per_vec != 0) return Q6_ERR_INVALID_ARGUMENT;
    if ((flags & ~Q6_NORM_ONE_PLUS) != 0) return Q6_ERR_INVALID_ARGUMENT;
    if (ldx < D && M > 1) return Q6_ERR_INVALID_ARGUMENT;
    if (has_vec && ldv < D && M > rows_per_vec) return Q6_ERR_INVALID_ARGUMENT;
    return Q6_OK;
}

bool aligned_to(const void* p, int dtype) {
    return reinterpret_cast<uintptr_t>(p) % (dtype == Q6_DTYPE_F32 ? 4 : 2) == 0;
}

}  // namespace
}  // namespace q6

extern "C" {

int q6_layer_norm(const void* x, int64_t ldx, const void* weight, const void* bias, int64_t ldv, int64_t rows_per_vec,
                  void* y, float* mean, float* rstd, int64_t M, int64_t D, float eps, int dtype, int vec_dtype,
                  int flags, q6_stream_t stream) {
    using namespace q6;
    const int st = check_norm(x, ldx, ldv, rows_per_vec, M, D, dtype, vec_dtype, flags, weight || bias);
    if (st != Q6_OK) return st;
    if (!y || (mean == nullptr) != (rstd == nullptr) || !(eps >= 0.0f)) return Q6_ERR_INVALID_ARGUMENT;
    if (!aligned_to(x, dtype) || !aligned_to(y, dtype) || !aligned_to(weight, vec_dtype) ||
        !aligned_to(bias, vec_dtype) || !aligned_to(mean, Q6_DTYPE_F32) || !aligned_to(rstd, Q6_DTYPE_F32))
        return Q6_ERR_ALIGNMENT;
    NormParams p{};
    p.x = x;
    p.ldx = ldx;
    p.weight = weight;
    p.bias = bias;
    p.ldv = ldv;
    p.rows_per_vec = rows_per_vec;
    p.y = y;
    p.mean = mean;
    p.rstd = rstd;
    p.M = M;
    p.D = D;
    p.eps = eps;
    p.one = (flags & Q6_NORM_ONE_PLUS) ? 1.0f : 0.0f;
    return with_types(dtype, vec_dtype, [&](auto t, auto v) {
        return run_forward<decltype(t), decltype(v)>(p, reinterpret_cast<cudaStream_t>(stream));
    });
}

size_t q6_layer_norm_grad_workspace_bytes(int64_t M, int64_t D, int64_t rows_per_vec, int dtype, int outputs) {
    (void)dtype;
    if (M <= 0 || D <= 0 || rows_per_vec <= 0 || M % rows_per_vec != 0) return 0;
    return q6::grad_bytes(M, D, rows_per_vec, outputs);
}

int q6_layer_norm_grad(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* weight, int64_t ldv,
                       int64_t rows_per_vec, const float* mean, const float* rstd, void* dx, void* dweight,
                       void* dbias, int64_t M, int64_t D, int dtype, int vec_dtype, int flags, void* workspace,
                       size_t workspace_bytes, q6_stream_t stream) {
    using namespace q6;
    const int st = check_norm(x, ldx, ldv, rows_per_vec, M, D, dtype, vec_dtype, flags, weight != nullptr);
    if (st != Q6_OK) return st;
    if (!dy || !mean || !rstd || (ldy < D && M > 1)) return Q6_ERR_INVALID_ARGUMENT;
    if (!aligned_to(x, dtype) || !aligned_to(dy, dtype) || !aligned_to(dx, dtype) || !aligned_to(weight, vec_dtype) ||
        !aligned_to(dweight, vec_dtype) || !aligned_to(dbias, vec_dtype) || !aligned_to(mean, Q6_DTYPE_F32) ||
        !aligned_to(rstd, Q6_DTYPE_F32))
        return Q6_ERR_ALIGNMENT;
    const int outputs = (dweight ? Q6_GRAD_W : 0) | (dbias ? Q6_GRAD_BIAS : 0);
    if (!dx && !outputs) return Q6_OK;
    if (workspace && reinterpret_cast<uintptr_t>(workspace) % 256) return Q6_ERR_ALIGNMENT;
    if (grad_bytes(M, D, rows_per_vec, outputs) > (workspace ? workspace_bytes : 0)) return Q6_ERR_WORKSPACE;
    NormParams p{};
    p.x = x;
    p.ldx = ldx;
    p.weight = weight;
    p.ldv = ldv;
    p.rows_per_vec = rows_per_vec;
    p.mean = const_cast<float*>(mean);
    p.rstd = const_cast<float*>(rstd);
    p.M = M;
    p.D = D;
    p.one = (flags & Q6_NORM_ONE_PLUS) ? 1.0f : 0.0f;
    p.dy = dy;
    p.ldy = ldy;
    p.dx = dx;
    plan_strips(M, rows_per_vec, &p.strip_rows, &p.strips_per_vec);
    p.col_blocks = static_cast<unsigned>((D + kThreads - 1) / kThreads);
    const size_t part = round_up(size_t(M / rows_per_vec) * p.strips_per_vec * D * sizeof(float));
    char* ws = static_cast<char*>(workspace);
    if (dweight) p.dw_part = reinterpret_cast<float*>(ws);
    if (dbias) p.db_part = reinterpret_cast<float*>(ws + (dweight ? part : 0));
    return with_types(dtype, vec_dtype, [&](auto t, auto v) {
        return run_grad<decltype(t), decltype(v)>(p, dweight, dbias, reinterpret_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
