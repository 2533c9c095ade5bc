// Dense 16-bit linear, forward and gradients (q6_dense_linear,
// q6_dense_linear_grad): the entry points, the aligned copies of operands the
// tensor core path cannot read in place, and the elementwise half of the
// backward pass.  The three products (x W^T, dz W, dz^T x) are
// launch_dense_product calls (q6_dense_gemm.cu).
//
// Backward, elementwise: with t = dy * gate,
//   dz = t act'(z),   dbias = sum_m dz,   dgate[s] = sum_{m in s} dy act(z).
// One pass reads dy and z once, writes dz (rounded to 16 bits, the operand of
// both products: with the output's own rounding that makes dx and dW 1.41 times one
// rounding's error; two 16-bit terms would avoid it at twice the tensor work) and
// sums its columns in fp32 from the unrounded values; each
// block sums a strip of rows of one sample, and a second small kernel adds the
// strips' partial sums in row order.  Nothing is accumulated with atomics, so
// equal calls give equal bits.
#include <algorithm>
#include <cstdint>
#include <cstdlib>

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

// Up to two operands [rows, cols] copied to row stride ldd, 16-bit elements; the
// pad columns are left alone (the tensor maps end at cols).  A block copies
// 2048 neighbouring columns of kPackRows rows, eight columns per thread and one
// 16-byte store for them.
struct PackOne {
    const uint16_t* src;
    uint16_t* dst;
    int64_t lds, ldd, rows, cols;
    unsigned col_blocks, blocks;
};
constexpr int kPackRows = 4;

__global__ void __launch_bounds__(256) pack_rows_kernel(const PackOne first, const PackOne second) {
    pdl_launch_dependents();
    pdl_wait();
    const bool one = blockIdx.x < first.blocks;
    const PackOne p = one ? first : second;
    const unsigned block = one ? blockIdx.x : blockIdx.x - first.blocks;
    const int64_t c0 = block % p.col_blocks * int64_t(2048) + threadIdx.x * 8;
    const int64_t r0 = block / p.col_blocks * int64_t(kPackRows);
    if (c0 >= p.cols) return;
    uint16_t v[kPackRows][8];
#pragma unroll
    for (int k = 0; k < kPackRows; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[k][i] = r0 + k < p.rows && c0 + i < p.cols ? __ldg(p.src + (r0 + k) * p.lds + c0 + i) : uint16_t(0);
#pragma unroll
    for (int k = 0; k < kPackRows; ++k)
        if (r0 + k < p.rows)
            *reinterpret_cast<uint4*>(p.dst + (r0 + k) * p.ldd + c0) =
                make_uint4(v[k][0] | uint32_t(v[k][1]) << 16, v[k][2] | uint32_t(v[k][3]) << 16,
                           v[k][4] | uint32_t(v[k][5]) << 16, v[k][6] | uint32_t(v[k][7]) << 16);
}

// The operands of one call that need an aligned copy (at most two).
struct Packer {
    PackOne part[2] = {};
    int n = 0;
    void add(const void* src, int64_t lds, void* dst, int64_t rows, int64_t cols) {
        PackOne& p = part[n++];
        p.src = static_cast<const uint16_t*>(src);
        p.dst = static_cast<uint16_t*>(dst);
        p.lds = lds;
        p.ldd = pad8(cols);
        p.rows = rows;
        p.cols = cols;
        p.col_blocks = static_cast<unsigned>((cols + 2047) / 2048);
        p.blocks = static_cast<unsigned>(std::min<int64_t>(p.col_blocks * ((rows + kPackRows - 1) / kPackRows), kMaxGrid));
    }
    int launch(cudaStream_t stream) const {
        if (n == 0) return Q6_OK;
        const int64_t blocks = int64_t(part[0].blocks) + part[1].blocks;
        if (blocks > kMaxGrid) return Q6_ERR_UNSUPPORTED;
        return launch_pdl(pack_rows_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, part[0],
                          part[1]) == cudaSuccess
                   ? Q6_OK
                   : Q6_ERR_CUDA;
    }
};

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
};

// A block takes 2048 neighbouring columns, eight per thread, and one strip of rows
// (all of one gate vector), kRows rows' loads in flight at a time.  kVec: 16-byte
// accesses (N, strides and addresses aligned); else single elements, a block's
// width apart.
//
// Bound by HBM (dy and z in, dz out): 3456 x 12288 with GELU 46 us of 39.5.  With
// twelve instructions per value for the activation in scalar form it was bound by
// issue (85 us), with two blocks per SM by the second wave (62 us).
template <typename T, typename Z, bool kVec, int ACT>
__global__ void __launch_bounds__(256, 3) dz_kernel(const DzParams p) {
    constexpr int kRows = 2;
    pdl_launch_dependents();
    pdl_wait();
    const int64_t col_block = blockIdx.x % p.col_blocks, strip = blockIdx.x / p.col_blocks;
    const int64_t s = strip / p.strips_per_gate;
    const int64_t r_begin = s * p.rows_per_gate + strip % p.strips_per_gate * p.strip_rows;
    const int rows = static_cast<int>(min(p.strip_rows, (s + 1) * p.rows_per_gate - r_begin));
    const int64_t c0 = col_block * 2048 + (kVec ? threadIdx.x * 8 : threadIdx.x);  // first column
    if (c0 >= p.N) return;
    const int left = static_cast<int>(min(p.N - c0, int64_t(2048)));  // strided: columns from c0 on in the block
    auto load = [&](auto* row) {
        using S = std::remove_cv_t<std::remove_pointer_t<decltype(row)>>;
        Group<S, 8> g;
        if constexpr (kVec) {
            g = load_ro<Group<S, 8>>(row);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) g.v[i] = 256 * i < left ? load_ro<S>(row + 256 * i) : from_f<S>(0.0f);
        }
        return g;
    };
    const T* dy = static_cast<const T*>(p.dy) + r_begin * p.ldy + c0;
    const Z* z = p.z ? static_cast<const Z*>(p.z) + r_begin * p.N + c0 : nullptr;
    T* dz = p.dz ? static_cast<T*>(p.dz) + r_begin * p.ldz + c0 : nullptr;
    float2 gate[4], db[4], dg[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        gate[i] = both(1.0f);
        db[i] = dg[i] = both(0.0f);
    }
    if (p.gate) unpack(load(static_cast<const T*>(p.gate) + s * p.ldg + c0), gate);
    for (int r0 = 0; r0 < rows; r0 += kRows) {
        Group<T, 8> gy[kRows];
        Group<Z, 8> gz[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int64_t r = min(r0 + k, rows - 1);  // past the end: the last row again, not used
            gy[k] = load(dy + r * p.ldy);
            if (z) gz[k] = load(z + r * p.N);
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            if (r0 + k < rows) {
                float2 fy[4], fz[4];
                unpack(gy[k], fy);
                if (z) unpack(gz[k], fz);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 d = mul2(fy[i], gate[i]);
                    if (z) {
                        float2 a, slope;
                        act_and_slope2<ACT>(fz[i], a, slope);
                        dg[i] = fma2(fy[i], a, dg[i]);
                        d = mul2(d, slope);
                    }
                    db[i] = add2(db[i], d);
                    fy[i] = d;
                }
                if (dz) {
                    const Group<T, 8> out = pack<T, 8>(fy);
                    T* to = dz + int64_t(r0 + k) * p.ldz;
                    if constexpr (kVec) {
                        *reinterpret_cast<Group<T, 8>*>(to) = out;
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (256 * i < left) to[256 * i] = out.v[i];
                    }
                }
            }
        }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* part = which == 0 ? p.db_part : p.dg_part;
        if (!part) continue;
        part += strip * p.N + c0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = which == 0 ? db[i / 2] : dg[i / 2];
            if (kVec || 256 * i < left) part[kVec ? i : 256 * i] = i & 1 ? v.y : v.x;
        }
    }
}

// dbias[n] = sum over all strips, dgate[g, n] = sum over gate vector g's strips, of
// the strips' partial sums, in order: 32 columns x 8 strip lanes per block.  The
// first db_blocks blocks sum dbias (none without it), the others dgate.
template <typename T>
__global__ void __launch_bounds__(256) sum_strips_kernel(const float* db_part, const float* dg_part, int64_t strips,
                                                         int64_t strips_per_gate, int64_t N, unsigned db_blocks,
                                                         T* dbias, T* dgate) {
    __shared__ float sum[8][33];
    pdl_launch_dependents();
    pdl_wait();
    const bool is_db = blockIdx.x < db_blocks;
    const unsigned block = is_db ? blockIdx.x : blockIdx.x - db_blocks;
    const unsigned col_blocks = static_cast<unsigned>((N + 31) / 32);
    const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int64_t n = block % col_blocks * int64_t(32) + cl, group = block / col_blocks;
    const int64_t count = is_db ? strips : strips_per_gate;
    const float* part = (is_db ? db_part : dg_part) + group * count * N;
    float t = 0.0f;
    if (n < N)
        for (int64_t i = sl; i < count; i += 80) {
            float f[10];
#pragma unroll
            for (int k = 0; k < 10; ++k) f[k] = i + 8 * k < count ? __ldcg(part + (i + 8 * k) * N + n) : 0.0f;
#pragma unroll
            for (int k = 0; k < 10; ++k) t += f[k];
        }
    sum[sl][cl] = t;
    __syncthreads();
    if (sl == 0 && n < N) {
#pragma unroll
        for (int i = 1; i < 8; ++i) t += sum[i][cl];
        (is_db ? dbias : dgate)[group * N + n] = from_f<T>(t);
    }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Rows per strip: one wave of three blocks per SM, strips of 4 rows at least.
void plan_strips(int64_t M, int64_t N, int64_t rows_per_gate, int64_t* strip_rows, int64_t* strips_per_gate) {
    const int64_t blocks = (N + 2047) / 2048 * (M / rows_per_gate);
    const int64_t want = std::max<int64_t>(1, int64_t(device_sm_count()) * 3 / blocks);
    *strip_rows = std::min(rows_per_gate, std::max<int64_t>(4, (rows_per_gate + want - 1) / want));
    *strips_per_gate = (rows_per_gate + *strip_rows - 1) / *strip_rows;
}

template <typename T, typename Z, int ACT>
int run_dz(DzParams p, int64_t M, void* dbias, void* dgate, cudaStream_t stream) {
    const int64_t gates = M / p.rows_per_gate, strips = gates * p.strips_per_gate;
    const bool vec = p.N % 8 == 0 && p.ldy % 8 == 0 && (!p.gate || p.ldg % 8 == 0) && aligned16(p.dy) &&
                     aligned16(p.z) && aligned16(p.gate);
    p.col_blocks = static_cast<unsigned>((p.N + 2047) / 2048);
    const int64_t db_blocks = dbias ? (p.N + 31) / 32 : 0, dg_blocks = dgate ? gates * ((p.N + 31) / 32) : 0;
    if (strips * p.col_blocks > kMaxGrid || db_blocks + dg_blocks > kMaxGrid) return Q6_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(strips * p.col_blocks));
    const cudaError_t e = vec ? launch_pdl(dz_kernel<T, Z, true, ACT>, grid, dim3(256), 0, stream, p)
                              : launch_pdl(dz_kernel<T, Z, false, ACT>, grid, dim3(256), 0, stream, p);
    if (e != cudaSuccess) return Q6_ERR_CUDA;
    if (db_blocks + dg_blocks == 0) return Q6_OK;
    return launch_pdl(sum_strips_kernel<T>, dim3(static_cast<unsigned>(db_blocks + dg_blocks)), dim3(256), 0, stream,
                      static_cast<const float*>(p.db_part), static_cast<const float*>(p.dg_part), strips,
                      p.strips_per_gate, p.N, static_cast<unsigned>(db_blocks), static_cast<T*>(dbias),
                      static_cast<T*>(dgate)) == cudaSuccess
               ? Q6_OK
               : Q6_ERR_CUDA;
}

template <typename T, typename Z>
int run_dz_act(const DzParams& p, int activation, int64_t M, void* dbias, void* dgate, cudaStream_t stream) {
    switch (activation) {
        case Q6_ACT_GELU_TANH: return run_dz<T, Z, Q6_ACT_GELU_TANH>(p, M, dbias, dgate, stream);
        case Q6_ACT_SILU: return run_dz<T, Z, Q6_ACT_SILU>(p, M, dbias, dgate, stream);
        default: return run_dz<T, Z, Q6_ACT_NONE>(p, M, dbias, dgate, stream);
    }
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

// The few-row kernel reads its operands where they are; Q6_DENSE_PLAN (a plan of
// the tensor-core path) turns it off.
bool few_rows(int64_t M, int64_t N, int64_t K) { return dense_few_rows(M, N, K) && !std::getenv("Q6_DENSE_PLAN"); }

size_t forward_bytes(int64_t M, int64_t N, int64_t K, int pack) {
    if (few_rows(M, N, K)) return 0;
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
    if (preact && preact_dtype != Q6_DTYPE_F16 && preact_dtype != Q6_DTYPE_F32) return Q6_ERR_UNSUPPORTED;
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
    DenseProduct a{};
    a.p_t = false;
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
    const bool rows = few_rows(M, N, K);
    Carver ws{static_cast<char*>(workspace)};
    if (!rows) {
        a.workspace_bytes = dense_product_workspace_bytes(M, N, K, false, false);
        a.workspace = ws.take(a.workspace_bytes);
        Packer packer;
        if (pack & Q6_PACK_X) {
            void* c = ws.take(size_t(M) * pad8(K) * 2);
            packer.add(x, ldx, c, M, K);
            x = c;
            ldx = pad8(K);
        }
        if (pack & Q6_PACK_W) {
            void* c = ws.take(size_t(N) * pad8(K) * 2);
            packer.add(w, ldw, c, N, K);
            w = c;
            ldw = pad8(K);
        }
        if (const int e = packer.launch(stream)) return e;
    }
    a.p = w;
    a.ldp = ldw;
    a.q = x;
    a.ldq = ldx;
    if (rows) return launch_dense_rows(a, stream);
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
    if (preact && preact_dtype != Q6_DTYPE_F16 && preact_dtype != Q6_DTYPE_F32) return Q6_ERR_UNSUPPORTED;
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
        int e;
        if (dtype == Q6_DTYPE_BF16)
            e = f32 ? run_dz_act<__nv_bfloat16, float>(z, activation, M, dbias, dgate, stream)
                    : run_dz_act<__nv_bfloat16, __half>(z, activation, M, dbias, dgate, stream);
        else
            e = f32 ? run_dz_act<__half, float>(z, activation, M, dbias, dgate, stream)
                    : run_dz_act<__half, __half>(z, activation, M, dbias, dgate, stream);
        if (e != Q6_OK) return e;
    }
    const void* t = wants_dz ? z.dz : dy;
    const int64_t ldt = wants_dz ? z.ldz : ldy;
    Packer packer;
    if (dx && (pack & Q6_PACK_W)) {
        void* c = ws.take(size_t(N) * pad8(K) * 2);
        packer.add(w, ldw, c, N, K);
        w = c;
        ldw = pad8(K);
    }
    if (dw && (pack & Q6_PACK_X)) {
        void* c = ws.take(size_t(M) * pad8(K) * 2);
        packer.add(x, ldx, c, M, K);
        x = c;
        ldx = pad8(K);
    }
    if (const int e = packer.launch(stream)) return e;
    if (dx) {
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
