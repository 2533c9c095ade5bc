// Layer norm entry points (q6_layer_norm, q6_layer_norm_grad), the plain kernels
// for rows wider than the register kernels hold (q6_norm.cuh), and the sums over
// strips.
#include "q6_norm.cuh"

namespace q6 {

void norm_plan_strips(int64_t M, int64_t rows_per_vec, int64_t least, int64_t* strip_rows, int64_t* strips_per_vec) {
    const int64_t vecs = M / rows_per_vec, per = std::max<int64_t>(1, device_sm_count() / vecs);
    *strip_rows = std::max<int64_t>(least, (rows_per_vec + per - 1) / per);
    *strips_per_vec = (rows_per_vec + *strip_rows - 1) / *strip_rows;
}

#define Q6_NORM_DECLARE(T, V)                                                                                        \
    template <>                                                                                                      \
    int norm_forward_typed<T, V>(const NormParams& p, bool vec, int shape, cudaStream_t stream);                     \
    template <>                                                                                                      \
    int norm_grad_typed<T, V>(const NormParams& p, bool vec, int shape, V* dweight, V* dbias, cudaStream_t stream);
Q6_NORM_DECLARE(__nv_bfloat16, __nv_bfloat16)
Q6_NORM_DECLARE(__nv_bfloat16, float)
Q6_NORM_DECLARE(__half, __half)
Q6_NORM_DECLARE(__half, float)
Q6_NORM_DECLARE(float, float)
#undef Q6_NORM_DECLARE

namespace {

constexpr int kThreads = 256;

// Plain kernels for rows that do not fit the registers: any width, stride and
// alignment.
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
template <typename T, typename V>
__global__ void __launch_bounds__(kThreads) norm_column_sums_kernel(NormParams p, V* dweight, V* dbias) {
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
    if (dweight) dweight[strip * p.D + c] = from_f<V>(dw);
    if (dbias) dbias[strip * p.D + c] = from_f<V>(db);
}

// out[v, c] = sum over vector v's strips of part[strip, c], in order: 32
// columns x 16 strip lanes per block, ten strips' loads in flight (a strip per
// SM: one round trip).  The first half of the grid sums dweight, the second
// dbias (either may be absent).
template <typename V>
__global__ void __launch_bounds__(512) norm_sum_strips_kernel(const float* dw_part, const float* db_part,
                                                              int64_t strips_per_vec, int64_t D, V* dweight,
                                                              V* dbias) {
    __shared__ float sum[16][33];
    pdl_launch_dependents();
    const unsigned half = gridDim.x / 2;
    const bool first = blockIdx.x < half;
    const unsigned block = first ? blockIdx.x : blockIdx.x - half;
    const float* part = first ? dw_part : db_part;
    V* out = first ? dweight : dbias;
    const unsigned col_blocks = static_cast<unsigned>((D + 31) / 32);
    const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int64_t c = block % col_blocks * int64_t(32) + cl, v = block / col_blocks;
    pdl_wait();
    if (!part) return;
    float t = 0.0f;
    if (c < D) {
        const float* src = part + v * strips_per_vec * D + c;
        for (int64_t i = sl; i < strips_per_vec; i += 160) {
            float f[10];
#pragma unroll
            for (int k = 0; k < 10; ++k) f[k] = i + 16 * k < strips_per_vec ? __ldcg(src + (i + 16 * k) * D) : 0.0f;
#pragma unroll
            for (int k = 0; k < 10; ++k) t += f[k];
        }
    }
    sum[sl][cl] = t;
    __syncthreads();
    if (sl == 0 && c < D) {
#pragma unroll
        for (int i = 1; i < 16; ++i) t += sum[i][cl];
        out[v * D + c] = from_f<V>(t);
    }
}

// The plain kernels sum columns with one thread each: more, shorter strips.
void plan_plain_strips(int64_t M, int64_t rows_per_vec, int64_t* strip_rows, int64_t* strips_per_vec) {
    const int64_t vecs = M / rows_per_vec, per = std::max<int64_t>(1, 4 * device_sm_count() / vecs);
    *strip_rows = (rows_per_vec + per - 1) / per;
    *strips_per_vec = (rows_per_vec + *strip_rows - 1) / *strip_rows;
}

size_t round_up(size_t v) { return (v + 255) / 256 * 256; }

// The backward's shape for a row of D (an index into kNormGrad or, without 16-byte
// accesses, kNormGradStrided; -1: the plain kernels) and its strips.
int plan_grad(int64_t M, int64_t D, int64_t rows_per_vec, int dtype, bool vec, int64_t* strip_rows,
              int64_t* strips_per_vec) {
    const int shape = vec ? norm_shape(kNormGrad, D, dtype) : norm_shape(kNormGradStrided, D, dtype);
    if (shape < 0)
        plan_plain_strips(M, rows_per_vec, strip_rows, strips_per_vec);
    else
        norm_plan_strips(M, rows_per_vec,
                         vec ? norm_detail::grad_row_lanes(kNormGrad[shape].w)
                             : strided_row_lanes(kNormGradStrided[shape].w),
                         strip_rows, strips_per_vec);
    return shape;
}

// Bytes of one vector gradient's partial sums, for either access width (none where
// a strip is a vector).
size_t part_bytes(int64_t M, int64_t D, int64_t rows_per_vec, int dtype) {
    int64_t rows, per, most = 1;
    for (const bool vec : {true, false}) {
        plan_grad(M, D, rows_per_vec, dtype, vec, &rows, &per);
        most = std::max(most, per);
    }
    return most == 1 ? 0 : round_up(size_t(M / rows_per_vec) * most * D * sizeof(float));
}

size_t grad_bytes(int64_t M, int64_t D, int64_t rows_per_vec, int dtype, int outputs) {
    const size_t part = part_bytes(M, D, rows_per_vec, dtype);
    return ((outputs & Q6_GRAD_W) ? part : 0) + ((outputs & Q6_GRAD_BIAS) ? part : 0);
}

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// 16-byte accesses to every operand: G elements of T, and of V in 16-byte parts.
template <typename T, typename V>
bool vector_ok(const NormParams& p) {
    constexpr int64_t G = 16 / sizeof(T);
    if (p.D % G || p.ldx % G || !al16(p.x) || !al16(p.weight) || !al16(p.bias)) return false;
    if ((p.weight || p.bias) && p.rows_per_vec < p.M && p.ldv * sizeof(V) % 16) return false;
    if (p.dy && (p.ldy % G || !al16(p.dy))) return false;
    return al16(p.y) && al16(p.dx);
}

template <typename T, typename V>
int run_forward(NormParams p, cudaStream_t stream) {
    const int shape = norm_shape(kNormForward, p.D, sizeof(T) == 4 ? Q6_DTYPE_F32 : Q6_DTYPE_BF16);
    if (shape >= 0) {
        const int64_t vecs = p.M / p.rows_per_vec;
        p.vecs = vecs > 1 && vecs <= 65535 ? static_cast<unsigned>(vecs) : 0;
        return norm_forward_typed<T, V>(p, vector_ok<T, V>(p), shape, stream);
    }
    return launch_pdl(norm_rows_kernel<T, V>, dim3(static_cast<unsigned>(p.M)), dim3(kThreads), 0, stream, p) ==
                   cudaSuccess
               ? Q6_OK
               : Q6_ERR_CUDA;
}

template <typename V>
int sum_strips(const NormParams& p, void* dweight, void* dbias, cudaStream_t stream) {
    const int64_t blocks = p.M / p.rows_per_vec * ((p.D + 31) / 32);
    if (2 * blocks > kNormMaxGrid) return Q6_ERR_UNSUPPORTED;
    return launch_pdl(norm_sum_strips_kernel<V>, dim3(static_cast<unsigned>(2 * blocks)), dim3(512), 0, stream,
                      static_cast<const float*>(p.dw_part), static_cast<const float*>(p.db_part), p.strips_per_vec,
                      p.D, static_cast<V*>(dweight), static_cast<V*>(dbias)) == cudaSuccess
               ? Q6_OK
               : Q6_ERR_CUDA;
}

template <typename T, typename V>
int run_grad(NormParams p, void* dweight, void* dbias, cudaStream_t stream) {
    const bool vec = vector_ok<T, V>(p);
    const int shape = plan_grad(p.M, p.D, p.rows_per_vec, sizeof(T) == 4 ? Q6_DTYPE_F32 : Q6_DTYPE_BF16, vec,
                                &p.strip_rows, &p.strips_per_vec);
    if (shape >= 0) {
        if (p.M / p.rows_per_vec * p.strips_per_vec > kNormMaxGrid) return Q6_ERR_UNSUPPORTED;
        const bool whole = p.strips_per_vec == 1;  // a strip is a vector: its sums are the result
        if (whole) p.dw_part = p.db_part = nullptr;
        const int st = norm_grad_typed<T, V>(p, vec, shape, whole ? static_cast<V*>(dweight) : static_cast<V*>(nullptr),
                                             whole ? static_cast<V*>(dbias) : static_cast<V*>(nullptr), stream);
        return st != Q6_OK || whole || (!dweight && !dbias) ? st : sum_strips<V>(p, dweight, dbias, stream);
    }
    if (p.dx && launch_pdl(norm_rows_dx_kernel<T, V>, dim3(static_cast<unsigned>(p.M)), dim3(kThreads), 0, stream,
                           static_cast<const NormParams>(p)) != cudaSuccess)
        return Q6_ERR_CUDA;
    if (!dweight && !dbias) return Q6_OK;
    const int64_t strips = p.M / p.rows_per_vec * p.strips_per_vec;
    p.col_blocks = static_cast<unsigned>((p.D + kThreads - 1) / kThreads);
    if (strips * p.col_blocks > kNormMaxGrid) return Q6_ERR_UNSUPPORTED;
    const bool whole = p.strips_per_vec == 1;
    if (whole) p.dw_part = p.db_part = nullptr;
    if (launch_pdl(norm_column_sums_kernel<T, V>, dim3(static_cast<unsigned>(strips * p.col_blocks)), dim3(kThreads), 0,
                   stream, static_cast<const NormParams>(p), whole ? static_cast<V*>(dweight) : static_cast<V*>(nullptr),
                   whole ? static_cast<V*>(dbias) : static_cast<V*>(nullptr)) != cudaSuccess)
        return Q6_ERR_CUDA;
    return whole ? Q6_OK : sum_strips<V>(p, dweight, dbias, stream);
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
    if (!x || M <= 0 || D <= 0 || M > kNormMaxGrid || D > (int64_t(1) << 30)) return Q6_ERR_INVALID_ARGUMENT;
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

int error_word_norm(bool clear) {
    int code = 0;
    for (const int w : {error_word_norm_bf16(clear), error_word_norm_f16(clear), error_word_norm_f32(clear)}) {
        if (w < 0) return -1;
        if (code == 0) code = w;
    }
    return code;
}

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
    p.inv = 1.0f / static_cast<float>(D);
    p.inv_rest = static_cast<float>(1.0 / static_cast<double>(D) - static_cast<double>(p.inv));
    p.one = (flags & Q6_NORM_ONE_PLUS) ? 1.0f : 0.0f;
    return with_types(dtype, vec_dtype, [&](auto t, auto v) {
        return run_forward<decltype(t), decltype(v)>(p, reinterpret_cast<cudaStream_t>(stream));
    });
}

size_t q6_layer_norm_grad_workspace_bytes(int64_t M, int64_t D, int64_t rows_per_vec, int dtype, int outputs) {
    if (M <= 0 || D <= 0 || rows_per_vec <= 0 || M % rows_per_vec != 0) return 0;
    return q6::grad_bytes(M, D, rows_per_vec, dtype, outputs);
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
    if (grad_bytes(M, D, rows_per_vec, dtype, outputs) > (workspace ? workspace_bytes : 0)) return Q6_ERR_WORKSPACE;
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
    const size_t part = part_bytes(M, D, rows_per_vec, dtype);
    char* ws = static_cast<char*>(workspace);
    if (dweight) p.dw_part = reinterpret_cast<float*>(ws);
    if (dbias) p.db_part = reinterpret_cast<float*>(ws + (dweight ? part : 0));
    return with_types(dtype, vec_dtype, [&](auto t, auto v) {
        return run_grad<decltype(t), decltype(v)>(p, dweight, dbias, reinterpret_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
