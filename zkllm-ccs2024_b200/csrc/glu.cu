// The gated feed-forward block up to its product: h = act(x Wg) * (x Wu), and the gradients of x, Wg and Wu.
//
// Weights are [in, hidden], as zkFC and FrTensor::matmul take them.  Sums are in 32 bits; h is formed from the unrounded sums.
#include <algorithm>

#include "floatops.cuh"

namespace zkb {
namespace {

// act(g) and, for the gradient, its derivative
template <bool kDerivative>
__device__ __forceinline__ float activate(int kind, float g, float* d) {
    if (kind == ZKB_ACT_SILU) {
        const float s = 1.0f / (1.0f + __expf(-g));
        if (kDerivative) *d = s * (1.0f + g * (1.0f - s));
        return g * s;
    }
    if (kind == ZKB_ACT_GELU) {
        const float c = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        if (kDerivative) *d = c + g * __expf(-0.5f * g * g) * 0.39894228040143268f;
        return g * c;
    }
    if (kind == ZKB_ACT_GELU_TANH) {
        // (1 + tanh k) / 2 = 1 / (1 + exp(-2k))
        const float k = 0.79788456080286536f * (g + 0.044715f * g * g * g);
        const float s = 1.0f / (1.0f + __expf(-2.0f * k));
        if (kDerivative) *d = s + 2.0f * g * s * (1.0f - s) * 0.79788456080286536f * (1.0f + 0.134145f * g * g);
        return g * s;
    }
    if (kDerivative) *d = g > 0.0f ? 1.0f : 0.0f;
    return fmaxf(g, 0.0f);
}

constexpr int kTile = 64, kDepth = 16;

// One 64 x 64 tile of sum_s A_s[m, k] B_s[k, n], any strides; 256 threads with 4 x 4 values each.
struct Product { const void *a, *b; size_t a_row, a_col, b_row, b_col; };
template <class T>
__device__ void tile_product(const Product& p, size_t M, size_t N, size_t K, float (&acc)[4][4]) {
    __shared__ float as[kDepth][kTile + 1], bs[kDepth][kTile + 1];
    const size_t m0 = (size_t)blockIdx.y * kTile, n0 = (size_t)blockIdx.x * kTile;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    for (size_t k0 = 0; k0 < K; k0 += kDepth) {
        for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
            const int m = p.a_col == 1 ? i / kDepth : i % kTile, k = p.a_col == 1 ? i % kDepth : i / kTile;
            as[k][m] = m0 + m < M && k0 + k < K ? to_f32<T>(static_cast<const T*>(p.a)[(m0 + m) * p.a_row + (k0 + k) * p.a_col]) : 0.0f;
            const int n = p.b_row == 1 ? i / kDepth : i % kTile, kb = p.b_row == 1 ? i % kDepth : i / kTile;
            bs[kb][n] = n0 + n < N && k0 + kb < K ? to_f32<T>(static_cast<const T*>(p.b)[(k0 + kb) * p.b_row + (n0 + n) * p.b_col]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += as[k][ty + 16 * i] * bs[k][tx + 16 * j];
        __syncthreads();
    }
}

template <class T>
__global__ void __launch_bounds__(256) glu_kernel(Product pg, Product pu, size_t M, size_t N, size_t K, T* h, size_t ldh, T* gate, size_t ldg, T* up,
                                                  size_t ldu, int act) {
    float g[4][4] = {}, u[4][4] = {};
    tile_product<T>(pg, M, N, K, g);
    tile_product<T>(pu, M, N, K, u);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const size_t m = (size_t)blockIdx.y * kTile + threadIdx.x / 16 + 16 * i, n = (size_t)blockIdx.x * kTile + threadIdx.x % 16 + 16 * j;
            if (m >= M || n >= N) continue;
            h[m * ldh + n] = from_f32<T>(activate<false>(act, g[i][j], nullptr) * u[i][j]);
            if (gate) gate[m * ldg + n] = from_f32<T>(g[i][j]);
            if (up) up[m * ldu + n] = from_f32<T>(u[i][j]);
        }
}

// one product, or the sum of two
template <class T>
__global__ void __launch_bounds__(256) glu_product_kernel(Product p0, Product p1, int products, size_t M, size_t N, size_t K, T* c, size_t ldc) {
    float acc[4][4] = {};
    tile_product<T>(p0, M, N, K, acc);
    if (products == 2) tile_product<T>(p1, M, N, K, acc);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const size_t m = (size_t)blockIdx.y * kTile + threadIdx.x / 16 + 16 * i, n = (size_t)blockIdx.x * kTile + threadIdx.x % 16 + 16 * j;
            if (m < M && n < N) c[m * ldc + n] = from_f32<T>(acc[i][j]);
        }
}

// The gradients of the two projections' results.  They are rounded to the tensors' type, as the operands of the products that
// follow have to be: each is off by half a step at most, independently, so a sum over them is off by no more, relative to its
// norm, than its own rounding.
template <class T>
__global__ void __launch_bounds__(256) glu_split_kernel(const T* gate, size_t ldg, const T* up, size_t ldu, const T* dh, size_t ldh, T* dg, T* du, size_t ld,
                                                        size_t rows, size_t cols, int act) {
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < rows * cols; i += (size_t)gridDim.x * 256) {
        const size_t m = i / cols, n = i % cols;
        const float g = to_f32<T>(gate[m * ldg + n]), u = to_f32<T>(up[m * ldu + n]), d = to_f32<T>(dh[m * ldh + n]);
        float da;
        const float a = activate<true>(act, g, &da);
        dg[m * ld + n] = from_f32<T>(d * u * da);
        du[m * ld + n] = from_f32<T>(d * a);
    }
}

struct GluArgs {
    int act;
    size_t tokens, in, hidden;
    const void *x, *wg, *wu, *gate, *up, *dh;
    size_t ldx, ldwg, ldwu, ldg, ldu, lddh;
    void *h, *gate_out, *up_out, *dx, *dwg, *dwu;
    size_t ldh, lddx, lddwg, lddwu;
};

template <class T>
int glu_launch(const GluArgs& a, cudaStream_t s) {
    const auto glu = glu_kernel<T>;
    ZKB_LAUNCH(glu, dim3(div_up(a.hidden, kTile), div_up(a.tokens, kTile)), 256, 0, s, Product{a.x, a.wg, a.ldx, 1, a.ldwg, 1},
               Product{a.x, a.wu, a.ldx, 1, a.ldwu, 1}, a.tokens, a.hidden, a.in, static_cast<T*>(a.h), a.ldh, static_cast<T*>(a.gate_out), a.ldg,
               static_cast<T*>(a.up_out), a.ldu, a.act);
    return ZKB_OK;
}

template <class T>
int glu_backward_launch(const GluArgs& a, cudaStream_t s) {
    Scratch scratch(s);
    T* dg = scratch.get_n<T>(a.tokens * a.hidden);
    T* du = scratch.get_n<T>(a.tokens * a.hidden);
    if (!dg || !du) return ZKB_ERR_CUDA;
    const auto glu_split = glu_split_kernel<T>;
    const auto glu_product = glu_product_kernel<T>;
    const size_t F = a.hidden;
    if (a.tokens && F)
        ZKB_LAUNCH(glu_split, (unsigned)std::min<size_t>(div_up(a.tokens * F, 256), 16 * sm_count()), 256, 0, s, static_cast<const T*>(a.gate), a.ldg,
                   static_cast<const T*>(a.up), a.ldu, static_cast<const T*>(a.dh), a.lddh, dg, du, F, a.tokens, F, a.act);
    if (a.dx && a.tokens)
        ZKB_LAUNCH(glu_product, dim3(div_up(a.in, kTile), div_up(a.tokens, kTile)), 256, 0, s, Product{dg, a.wg, F, 1, 1, a.ldwg},
                   Product{du, a.wu, F, 1, 1, a.ldwu}, 2, a.tokens, a.in, F, static_cast<T*>(a.dx), a.lddx);
    for (int k = 0; k < 2; ++k) {
        void* out = k ? a.dwu : a.dwg;
        if (!out || !F) continue;
        ZKB_LAUNCH(glu_product, dim3(div_up(F, kTile), div_up(a.in, kTile)), 256, 0, s, Product{a.x, k ? du : dg, 1, a.ldx, F, 1}, Product{}, 1, a.in, F,
                   a.tokens, static_cast<T*>(out), k ? a.lddwu : a.lddwg);
    }
    return ZKB_OK;
}

int check_matrix(const char* who, const char* name, const void* p, size_t rows, size_t cols, size_t ld, bool needed) {
    const std::string w = std::string(who) + ": " + name;
    if (!p) return needed ? fail(ZKB_ERR_ARG, w + " is missing") : ZKB_OK;
    if (ld < cols && rows > 1) return fail(ZKB_ERR_DIM, w + ": row stride below the row's length");
    return check_device(p, 2, w.c_str());
}
int check_common(const char* who, int dtype, int act, const GluArgs& a) {
    const std::string w(who);
    if (dtype != ZKB_F16 && dtype != ZKB_BF16) return fail(ZKB_ERR_ARG, w + ": f16 or bf16 is wanted");
    if (act < ZKB_ACT_SILU || act > ZKB_ACT_RELU) return fail(ZKB_ERR_ARG, w + ": unknown activation");
    if (a.tokens > (1u << 22) || a.in > (1u << 20) || a.hidden > (1u << 20))
        return fail(ZKB_ERR_LIMIT, w + ": more than 2^22 tokens or 2^20 channels");
    return ZKB_OK;
}

}  // namespace
}  // namespace zkb

using namespace zkb;

extern "C" {

int zkb_glu(int dtype, int activation, size_t tokens, size_t in_dim, size_t hidden, const void* d_x, size_t ldx, const void* d_w_gate, size_t ldwg,
            const void* d_w_up, size_t ldwu, void* d_h, size_t ldh, void* d_gate, size_t ldg, void* d_up, size_t ldu, void* stream) {
    ZKB_API_RANGE();
    const char* who = "zkb_glu";
    GluArgs a = {};
    a.act = activation;
    a.tokens = tokens, a.in = in_dim, a.hidden = hidden;
    a.x = d_x, a.ldx = ldx, a.wg = d_w_gate, a.ldwg = ldwg, a.wu = d_w_up, a.ldwu = ldwu;
    a.h = d_h, a.ldh = ldh, a.gate_out = d_gate, a.ldg = ldg, a.up_out = d_up, a.ldu = ldu;
    ZKB_TRY(check_common(who, dtype, activation, a));
    if (!d_gate != !d_up) return fail(ZKB_ERR_ARG, "zkb_glu: gate and up are kept together or not at all");
    if (!tokens || !hidden) return ZKB_OK;
    ZKB_TRY(check_matrix(who, "x", d_x, tokens, in_dim, ldx, in_dim != 0));
    ZKB_TRY(check_matrix(who, "w_gate", d_w_gate, in_dim, hidden, ldwg, in_dim != 0));
    ZKB_TRY(check_matrix(who, "w_up", d_w_up, in_dim, hidden, ldwu, in_dim != 0));
    ZKB_TRY(check_matrix(who, "h", d_h, tokens, hidden, ldh, true));
    ZKB_TRY(check_matrix(who, "gate", d_gate, tokens, hidden, ldg, false));
    ZKB_TRY(check_matrix(who, "up", d_up, tokens, hidden, ldu, false));
    const cudaStream_t s = as_stream(stream);
    return dtype == ZKB_F16 ? glu_launch<__half>(a, s) : glu_launch<bf16>(a, s);
}

int zkb_glu_backward(int dtype, int activation, size_t tokens, size_t in_dim, size_t hidden, const void* d_x, size_t ldx, const void* d_w_gate, size_t ldwg,
                     const void* d_w_up, size_t ldwu, const void* d_gate, size_t ldg, const void* d_up, size_t ldu, const void* d_dh, size_t lddh,
                     void* d_dx, size_t lddx, void* d_dw_gate, size_t lddwg, void* d_dw_up, size_t lddwu, void* stream) {
    ZKB_API_RANGE();
    const char* who = "zkb_glu_backward";
    GluArgs a = {};
    a.act = activation;
    a.tokens = tokens, a.in = in_dim, a.hidden = hidden;
    a.x = d_x, a.ldx = ldx, a.wg = d_w_gate, a.ldwg = ldwg, a.wu = d_w_up, a.ldwu = ldwu;
    a.gate = d_gate, a.ldg = ldg, a.up = d_up, a.ldu = ldu, a.dh = d_dh, a.lddh = lddh;
    a.dx = d_dx, a.lddx = lddx, a.dwg = d_dw_gate, a.lddwg = lddwg, a.dwu = d_dw_up, a.lddwu = lddwu;
    ZKB_TRY(check_common(who, dtype, activation, a));
    if (!d_dw_gate != !d_dw_up) return fail(ZKB_ERR_ARG, "zkb_glu_backward: both weights' gradients or none");
    if (!in_dim) return ZKB_OK;
    const bool some = tokens && hidden;
    ZKB_TRY(check_matrix(who, "x", d_x, tokens, in_dim, ldx, some && d_dw_gate));
    ZKB_TRY(check_matrix(who, "w_gate", d_w_gate, in_dim, hidden, ldwg, some && d_dx));
    ZKB_TRY(check_matrix(who, "w_up", d_w_up, in_dim, hidden, ldwu, some && d_dx));
    ZKB_TRY(check_matrix(who, "gate", d_gate, tokens, hidden, ldg, some));
    ZKB_TRY(check_matrix(who, "up", d_up, tokens, hidden, ldu, some));
    ZKB_TRY(check_matrix(who, "dh", d_dh, tokens, hidden, lddh, some));
    ZKB_TRY(check_matrix(who, "dx", d_dx, tokens, in_dim, lddx, false));
    ZKB_TRY(check_matrix(who, "dw_gate", d_dw_gate, in_dim, hidden, lddwg, false));
    ZKB_TRY(check_matrix(who, "dw_up", d_dw_up, in_dim, hidden, lddwu, false));
    const cudaStream_t s = as_stream(stream);
    return dtype == ZKB_F16 ? glu_backward_launch<__half>(a, s) : glu_backward_launch<bf16>(a, s);
}

}  // extern "C"
