// Dense 16-bit linear, forward and gradients (q6_dense_linear,
// q6_dense_linear_grad): the entry points, the aligned copies of operands the
// tensor core path cannot read in place, and the elementwise half of the
// backward pass.  The three products (x W^T, dz W, dz^T x) are
// launch_dense_product calls (q6_dense_gemm.cu).
//
// Backward, elementwise: with t = dy * gate,
//   dz = t act'(z),   dbias = sum_m dz,   dgate[s] = sum_{m in s} dy act(z).
// One pass reads dy and z once, writes dz (rounded to 16 bits, the operand of
// both products) and sums its columns in fp32 from the unrounded values; each
// block sums a strip of rows of one sample, and a second small kernel adds the
// strips' partial sums in row order.  Nothing is accumulated with atomics, so
// equal calls give equal bits.
#include <algorithm>
#include <cstdint>

#include "q6_dense.cuh"
#include "q6_dense.h"
#include "q6_internal.h"
#include "q6_ptx.cuh"

namespace q6 {
namespace {

constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;
constexpr size_t kAlign = 256;  // workspace parts start on 256-byte boundaries
size_t round_up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }
int64_t pad8(int64_t v) { return (v + 7) / 8 * 8; }

// ------------------------------------------------------------------- aligned copy

// dst [rows, cols] with row stride ldd from src with row stride lds, 16-bit
// elements; the pad columns of dst are left alone (the tensor maps end at cols).
__global__ void __launch_bounds__(256) pack_rows_kernel(const uint16_t* __restrict__ src, int64_t lds, uint16_t* dst,
                                                        int64_t ldd, int64_t rows, int64_t cols) {
    pdl_launch_dependents();
    pdl_wait();
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
        for (int64_t c = blockIdx.x * int64_t(256) + threadIdx.x; c < cols; c += int64_t(gridDim.x) * 256)
            dst[r * ldd + c] = src[r * lds + c];
}

int launch_pack(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols, cudaStream_t stream) {
    const unsigned gx = static_cast<unsigned>(std::min<int64_t>((cols + 255) / 256, 1024));
    const unsigned gy = static_cast<unsigned>(std::min<int64_t>(rows, std::max<int64_t>(1, 148 * 32 / gx)));
    return launch_pdl(pack_rows_kernel, dim3(gx, gy), dim3(256), 0, stream, static_cast<const uint16_t*>(src), lds,
                      static_cast<uint16_t*>(dst), ldd, rows, cols) == cudaSuccess
               ? Q6_OK
               : Q6_ERR_CUDA;
}

// ---------------------------------------------------------- elementwise backward

struct DzParams {
    const void* dy;
    int64_t ldy;
    const void* z;  // [M, N] dense, element type Z of the kernel, or null
    const void* gate;
    int64_t ldg;
    void* dz;  // row stride ldz, or null
    int64_t ldz;
    float* db_part;  // [strips, N] or null
    float* dg_part;  // [strips, N] or null
    int64_t N;
    int64_t rows_per_gate;
    int64_t strip_rows, strips_per_gate;
    unsigned col_blocks;
    int activation;
};

// A block takes 32 * V columns and one strip of rows (all of one gate vector):
// 32 column lanes x 8 row lanes.  V = 8: 16-byte accesses (N, strides and
// addresses aligned); V = 1: any layout.
template <typename T, typename Z, int V>
__global__ void __launch_bounds__(256) dz_kernel(DzParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int64_t col_block = blockIdx.x % p.col_blocks, strip = blockIdx.x / p.col_blocks;
    const int64_t c0 = (col_block * 32 + cl) * V;
    const int64_t s = strip / p.strips_per_gate;
    const int64_t r_end = std::min((s + 1) * p.rows_per_gate,
                                   s * p.rows_per_gate + (strip % p.strips_per_gate + 1) * p.strip_rows);
    int64_t r = s * p.rows_per_gate + (strip % p.strips_per_gate) * p.strip_rows + rl;
    const bool in = c0 < p.N;
    float gate[V], db[V], dg[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        gate[i] = in && p.gate ? to_f(static_cast<const T*>(p.gate)[s * p.ldg + c0 + i]) : 1.0f;
        db[i] = dg[i] = 0.0f;
    }
    struct alignas(sizeof(T) * V) Group {
        T v[V];
    };
    struct alignas(V == 8 ? 16 : sizeof(Z)) GroupZ {
        Z v[V];
    };
    if (in) {
#pragma unroll 2
        for (; r < r_end; r += 8) {
            const Group gy = *reinterpret_cast<const Group*>(static_cast<const T*>(p.dy) + r * p.ldy + c0);
            Group out;
            GroupZ gz;
            if (p.z) gz = *reinterpret_cast<const GroupZ*>(static_cast<const Z*>(p.z) + r * p.N + c0);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float dy = to_f(gy.v[i]);
                float a = 0.0f, slope = 1.0f;
                if (p.z) act_and_slope_f(to_f(gz.v[i]), p.activation, a, slope);
                const float dz = dy * gate[i] * slope;
                db[i] += dz;
                dg[i] = fmaf(dy, a, dg[i]);
                out.v[i] = from_f<T>(dz);
            }
            if (p.dz) *reinterpret_cast<Group*>(static_cast<T*>(p.dz) + r * p.ldz + c0) = out;
        }
    }
    // column sums over the eight row lanes, in order
    __shared__ float sum[8][32 * V];
    for (int pass = 0; pass < 2; ++pass) {
        float* part = pass == 0 ? p.db_part : p.dg_part;
        if (!part) continue;  // the same for the whole block
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) sum[rl][cl * V + i] = pass == 0 ? db[i] : dg[i];
        __syncthreads();
        for (int c = threadIdx.x; c < 32 * V; c += 256) {
            const int64_t col = col_block * (32 * V) + c;
            if (col < p.N) {
                float t = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) t += sum[k][c];
                part[strip * p.N + col] = t;
            }
        }
    }
}

// out[g, n] = sum over group g's strips of part[strip, n], in order.
template <typename T>
__global__ void __launch_bounds__(128) sum_strips_kernel(const float* __restrict__ part, int64_t strips_per_group,
                                                         int64_t N, T* out) {
    pdl_launch_dependents();
    pdl_wait();
    const unsigned col_blocks = static_cast<unsigned>((N + 127) / 128);
    const int64_t n = blockIdx.x % col_blocks * int64_t(128) + threadIdx.x, group = blockIdx.x / col_blocks;
    if (n >= N) return;
    const float* src = part + group * strips_per_group * N + n;
    float t = 0.0f;
#pragma unroll 8
    for (int64_t i = 0; i < strips_per_group; ++i) t += src[i * N];
    out[group * N + n] = from_f<T>(t);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Rows per strip: enough blocks for the GPU, strips of 32 rows at least.
void plan_strips(int64_t M, int64_t N, int64_t rows_per_gate, int64_t* strip_rows, int64_t* strips_per_gate) {
    const int64_t col_blocks = (N + 255) / 256, gates = M / rows_per_gate;
    const int64_t want = std::max<int64_t>(1, (148 * 4 + col_blocks * gates - 1) / (col_blocks * gates));
    int64_t rows = std::max<int64_t>(32, (rows_per_gate + want - 1) / want);
    rows = std::min(rows, rows_per_gate);
    *strip_rows = rows;
    *strips_per_gate = (rows_per_gate + rows - 1) / rows;
}

template <typename T, typename Z>
int run_dz(DzParams p, int64_t M, void* dbias, void* dgate, cudaStream_t stream) {
    const int64_t gates = M / p.rows_per_gate, strips = gates * p.strips_per_gate;
    const bool vec = p.N % 8 == 0 && p.ldy % 8 == 0 && (!p.gate || p.ldg % 8 == 0) && aligned16(p.dy) &&
                     aligned16(p.z) && aligned16(p.gate);
    const int cols = vec ? 256 : 32;
    p.col_blocks = static_cast<unsigned>((p.N + cols - 1) / cols);
    const int64_t sum_blocks = (p.N + 127) / 128;
    if (strips * p.col_blocks > kMaxGrid || gates * sum_blocks > kMaxGrid) return Q6_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(strips * p.col_blocks));
    const cudaError_t e = vec ? launch_pdl(dz_kernel<T, Z, 8>, grid, dim3(256), 0, stream, p)
                              : launch_pdl(dz_kernel<T, Z, 1>, grid, dim3(256), 0, stream, p);
    if (e != cudaSuccess) return Q6_ERR_CUDA;
    if (dbias && launch_pdl(sum_strips_kernel<T>, dim3(static_cast<unsigned>(sum_blocks)), dim3(128), 0, stream,
                            static_cast<const float*>(p.db_part), strips, p.N, static_cast<T*>(dbias)) != cudaSuccess)
        return Q6_ERR_CUDA;
    if (dgate && launch_pdl(sum_strips_kernel<T>, dim3(static_cast<unsigned>(gates * sum_blocks)), dim3(128), 0, stream,
                            static_cast<const float*>(p.dg_part), p.strips_per_gate, p.N,
                            static_cast<T*>(dgate)) != cudaSuccess)
        return Q6_ERR_CUDA;
    return Q6_OK;
}

constexpr int64_t kMaxDim = int64_t(1) << 30;

bool dims_ok(int64_t M, int64_t N, int64_t K) {
    return M > 0 && N > 0 && K > 0 && M <= kMaxDim && N <= kMaxDim && K <= kMaxDim;
}

bool needs_pack(const void* p, int64_t ld) { return !aligned16(p) || ld % 8 != 0; }

// Hands out 256-byte aligned parts of the caller's workspace.
struct Carver {
    char* base;
    size_t used = 0;
    void* take(size_t bytes) {
        const size_t at = used;
        used += round_up(bytes);
        return base ? base + at : nullptr;
    }
};

size_t forward_bytes(int64_t M, int64_t N, int64_t K, int pack) {
    size_t b = round_up(dense_product_workspace_bytes(M, N, K, false, false));
    if (pack & Q6_PACK_X) b += round_up(size_t(M) * pad8(K) * 2);
    if (pack & Q6_PACK_W) b += round_up(size_t(N) * pad8(K) * 2);
    return b;
}

bool writes_dz(int activation, int has_gate, int outputs, int pack) {
    return (outputs & (Q6_GRAD_X | Q6_GRAD_W)) && (activation != Q6_ACT_NONE || has_gate || (pack & Q6_PACK_DY));
}

size_t product_bytes_grad(int64_t M, int64_t N, int64_t K, int outputs) {
    size_t b = 0;
    if (outputs & Q6_GRAD_X) b = std::max(b, dense_product_workspace_bytes(M, K, N, true, false));
    if (outputs & Q6_GRAD_W) b = std::max(b, dense_product_workspace_bytes(N, K, M, true, true));
    return b;
}

size_t grad_bytes(int64_t M, int64_t N, int64_t K, int64_t rows_per_gate, int activation, int has_gate, int outputs,
                  int pack) {
    int64_t rows = 0, per = 0;
    plan_strips(M, N, rows_per_gate, &rows, &per);
    const size_t part = size_t(M / rows_per_gate) * per * N * sizeof(float);
    size_t b = round_up(product_bytes_grad(M, N, K, outputs));
    if (writes_dz(activation, has_gate, outputs, pack)) b += round_up(size_t(M) * pad8(N) * 2);
    if (outputs & Q6_GRAD_BIAS) b += round_up(part);
    if (outputs & Q6_GRAD_GATE) b += round_up(part);
    if ((pack & Q6_PACK_X) && (outputs & Q6_GRAD_W)) b += round_up(size_t(M) * pad8(K) * 2);
    if ((pack & Q6_PACK_W) && (outputs & Q6_GRAD_X)) b += round_up(size_t(N) * pad8(K) * 2);
    return b;
}

int check_common(int64_t M, int64_t N, int64_t K, int dtype, int activation, const void* gate, int64_t ldg,
                 int64_t rows_per_gate) {
    if (!dims_ok(M, N, K)) return Q6_ERR_INVALID_ARGUMENT;
    if (dtype != Q6_DTYPE_BF16 && dtype != Q6_DTYPE_F16) return Q6_ERR_UNSUPPORTED;
    if (activation < Q6_ACT_NONE || activation > Q6_ACT_SILU) return Q6_ERR_INVALID_ARGUMENT;
    if (rows_per_gate <= 0 || rows_per_gate > M || M % rows_per_gate != 0) return Q6_ERR_INVALID_ARGUMENT;
    if (gate && M > rows_per_gate && ldg < N) return Q6_ERR_INVALID_ARGUMENT;
    return Q6_OK;
}

bool stride_ok(int64_t ld, int64_t width, int64_t rows) { return ld >= width || rows == 1; }
bool element_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 2 == 0; }

}  // namespace
}  // namespace q6

extern "C" {

size_t q6_dense_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int pack) {
    return q6::dims_ok(M, N, K) ? q6::forward_bytes(M, N, K, pack) : 0;
}

size_t q6_dense_linear_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t rows_per_gate, int activation,
                                            int has_gate, int outputs, int pack) {
    if (!q6::dims_ok(M, N, K) || rows_per_gate <= 0 || M % rows_per_gate != 0) return 0;
    return q6::grad_bytes(M, N, K, rows_per_gate, activation, has_gate, outputs, pack);
}

int q6_dense_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* gate,
                    int64_t ldg, int64_t rows_per_gate, const void* residual, int64_t ldr, void* y, void* preact,
                    int preact_dtype, int64_t M, int64_t N, int64_t K, int dtype, int activation, void* workspace,
                    size_t workspace_bytes, q6_stream_t stream_) {
    using namespace q6;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    const int st = check_common(M, N, K, dtype, activation, gate, ldg, rows_per_gate);
    if (st != Q6_OK) return st;
    if (!x || !w || !y) return Q6_ERR_INVALID_ARGUMENT;
    if (preact && preact_dtype != dtype && preact_dtype != Q6_DTYPE_F32) return Q6_ERR_UNSUPPORTED;
    if (!stride_ok(ldx, K, M) || !stride_ok(ldw, K, N) || (residual && !stride_ok(ldr, N, M)))
        return Q6_ERR_INVALID_ARGUMENT;
    for (const void* t : {x, w, bias, gate, residual, static_cast<const void*>(y), static_cast<const void*>(preact)})
        if (!element_aligned(t)) return Q6_ERR_ALIGNMENT;
    if (preact && preact_dtype == Q6_DTYPE_F32 && reinterpret_cast<uintptr_t>(preact) % 4) return Q6_ERR_ALIGNMENT;
    if (M == 1) ldx = pad8(K);  // a single row has no stride
    if (N == 1) ldw = pad8(K);
    const int pack = (needs_pack(x, ldx) ? Q6_PACK_X : 0) | (needs_pack(w, ldw) ? Q6_PACK_W : 0);
    if (workspace && reinterpret_cast<uintptr_t>(workspace) % kAlign) return Q6_ERR_ALIGNMENT;
    const size_t need = forward_bytes(M, N, K, pack);
    if (need > (workspace ? workspace_bytes : 0)) return Q6_ERR_WORKSPACE;
    Carver ws{static_cast<char*>(workspace)};
    DenseProduct a{};
    a.workspace_bytes = dense_product_workspace_bytes(M, N, K, false, false);
    a.workspace = ws.take(a.workspace_bytes);
    if (pack & Q6_PACK_X) {
        void* c = ws.take(size_t(M) * pad8(K) * 2);
        if (const int e = launch_pack(x, ldx, c, pad8(K), M, K, stream)) return e;
        x = c;
        ldx = pad8(K);
    }
    if (pack & Q6_PACK_W) {
        void* c = ws.take(size_t(N) * pad8(K) * 2);
        if (const int e = launch_pack(w, ldw, c, pad8(K), N, K, stream)) return e;
        w = c;
        ldw = pad8(K);
    }
    a.p = w;
    a.ldp = ldw;
    a.p_t = false;
    a.q = x;
    a.ldq = ldx;
    a.q_t = false;
    a.d = y;
    a.R = M;
    a.C = N;
    a.L = K;
    a.dtype = dtype;
    a.epi.bias = bias;
    a.epi.gate = gate;
    a.epi.ldg = ldg;
    a.epi.rows_per_gate = rows_per_gate;
    a.epi.residual = residual;
    a.epi.ldr = ldr;
    a.epi.preact = preact;
    a.epi.preact_f32 = preact_dtype == Q6_DTYPE_F32;
    a.epi.activation = activation;
    return launch_dense_product(a, stream);
}

int q6_dense_linear_grad(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* w, int64_t ldw,
                         const void* preact, int preact_dtype, const void* gate, int64_t ldg, int64_t rows_per_gate,
                         void* dx, void* dw, void* dbias, void* dgate, int64_t M, int64_t N, int64_t K, int dtype,
                         int activation, void* workspace, size_t workspace_bytes, q6_stream_t stream_) {
    using namespace q6;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    const int st = check_common(M, N, K, dtype, activation, gate, ldg, rows_per_gate);
    if (st != Q6_OK) return st;
    if (!dy || (dw && !x) || (dx && !w)) return Q6_ERR_INVALID_ARGUMENT;
    if (!preact && (activation != Q6_ACT_NONE || dgate)) return Q6_ERR_INVALID_ARGUMENT;
    if (preact && preact_dtype != dtype && preact_dtype != Q6_DTYPE_F32) return Q6_ERR_UNSUPPORTED;
    if (dgate && !gate) return Q6_ERR_INVALID_ARGUMENT;
    if (!stride_ok(ldy, N, M) || (dw && !stride_ok(ldx, K, M)) || (dx && !stride_ok(ldw, K, N)))
        return Q6_ERR_INVALID_ARGUMENT;
    for (const void* t : {dy, x, w, preact, gate, static_cast<const void*>(dx), static_cast<const void*>(dw),
                          static_cast<const void*>(dbias), static_cast<const void*>(dgate)})
        if (!element_aligned(t)) return Q6_ERR_ALIGNMENT;
    const int outputs = (dx ? Q6_GRAD_X : 0) | (dw ? Q6_GRAD_W : 0) | (dbias ? Q6_GRAD_BIAS : 0) |
                        (dgate ? Q6_GRAD_GATE : 0);
    if (outputs == 0) return Q6_OK;
    if (preact && preact_dtype == Q6_DTYPE_F32 && reinterpret_cast<uintptr_t>(preact) % 4) return Q6_ERR_ALIGNMENT;
    if (M == 1) ldx = pad8(K), ldy = pad8(N);  // a single row has no stride
    if (N == 1) ldw = pad8(K);
    const int pack = (needs_pack(x, ldx) ? Q6_PACK_X : 0) | (needs_pack(w, ldw) ? Q6_PACK_W : 0) |
                     (needs_pack(dy, ldy) ? Q6_PACK_DY : 0);
    if (workspace && reinterpret_cast<uintptr_t>(workspace) % kAlign) return Q6_ERR_ALIGNMENT;
    const size_t need = grad_bytes(M, N, K, rows_per_gate, activation, gate != nullptr, outputs, pack);
    if (need > (workspace ? workspace_bytes : 0)) return Q6_ERR_WORKSPACE;
    Carver ws{static_cast<char*>(workspace)};
    const size_t product_bytes = product_bytes_grad(M, N, K, outputs);
    void* product_ws = ws.take(product_bytes);

    DzParams z{};
    z.dy = dy;
    z.ldy = ldy;
    z.z = (activation != Q6_ACT_NONE || dgate) ? preact : nullptr;
    z.gate = gate;
    z.ldg = ldg;
    z.N = N;
    z.rows_per_gate = rows_per_gate;
    z.activation = activation;
    plan_strips(M, N, rows_per_gate, &z.strip_rows, &z.strips_per_gate);
    const size_t part = size_t(M / rows_per_gate) * z.strips_per_gate * N * sizeof(float);
    const bool wants_dz = writes_dz(activation, gate != nullptr, outputs, pack);
    if (wants_dz) {
        z.ldz = pad8(N);
        z.dz = ws.take(size_t(M) * z.ldz * 2);
    }
    if (dbias) z.db_part = static_cast<float*>(ws.take(part));
    if (dgate) z.dg_part = static_cast<float*>(ws.take(part));
    if (wants_dz || dbias || dgate) {
        const bool f32 = z.z && preact_dtype == Q6_DTYPE_F32;
        const int e = dtype == Q6_DTYPE_BF16 ? (f32 ? run_dz<__nv_bfloat16, float>(z, M, dbias, dgate, stream)
                                                    : run_dz<__nv_bfloat16, __nv_bfloat16>(z, M, dbias, dgate, stream))
                                             : (f32 ? run_dz<__half, float>(z, M, dbias, dgate, stream)
                                                    : run_dz<__half, __half>(z, M, dbias, dgate, stream));
        if (e != Q6_OK) return e;
    }
    const void* t = wants_dz ? z.dz : dy;
    const int64_t ldt = wants_dz ? z.ldz : ldy;
    if (dx) {
        if (pack & Q6_PACK_W) {
            void* c = ws.take(size_t(N) * pad8(K) * 2);
            if (const int e = launch_pack(w, ldw, c, pad8(K), N, K, stream)) return e;
            w = c;
            ldw = pad8(K);
        }
        DenseProduct a{};  // dx[m, k] = sum_n dz[m, n] W[n, k]
        a.p = w;
        a.ldp = ldw;
        a.p_t = true;
        a.q = t;
        a.ldq = ldt;
        a.q_t = false;
        a.d = dx;
        a.R = M;
        a.C = K;
        a.L = N;
        a.dtype = dtype;
        a.workspace = product_ws;
        a.workspace_bytes = product_bytes;
        if (const int e = launch_dense_product(a, stream)) return e;
    }
    if (dw) {
        if (pack & Q6_PACK_X) {
            void* c = ws.take(size_t(M) * pad8(K) * 2);
            if (const int e = launch_pack(x, ldx, c, pad8(K), M, K, stream)) return e;
            x = c;
            ldx = pad8(K);
        }
        DenseProduct a{};  // dw[n, k] = sum_m dz[m, n] x[m, k]
        a.p = x;
        a.ldp = ldx;
        a.p_t = true;
        a.q = t;
        a.ldq = ldt;
        a.q_t = true;
        a.d = dw;
        a.R = N;
        a.C = K;
        a.L = M;
        a.dtype = dtype;
        a.workspace = product_ws;
        a.workspace_bytes = product_bytes;
        if (const int e = launch_dense_product(a, stream)) return e;
    }
    return Q6_OK;
}

}  // extern "C"
