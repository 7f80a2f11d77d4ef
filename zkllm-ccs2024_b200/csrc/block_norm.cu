// The norms after one branch of a layer and before the next, with the branch's gate, residual scale and addition between them.
//
//     n = y / sqrt(mean y^2 + eps) * w_post      (or y, without the norm after the branch)
//     r = x + a * gate * n
//     z = r / sqrt(mean r^2 + eps) * w_pre
//
// and the gradients of x, y, the gate and both gains.  Sums are in 32 bits; z is formed from r before r is rounded.
#include <algorithm>

#include "floatops.cuh"

namespace zkb {
namespace {

constexpr size_t kMaxCols = 16384;

struct NormArgs {
    size_t rows, cols;
    const void *x, *y, *gate, *post_gain, *pre_gain;
    size_t ldx, ldy, ldgate;
    void *r, *z;
    size_t ldr, ldz;
    float *post_inv, *pre_inv;
    float scale, eps;
    int gate_kind;
    bool post_norm, pre_norm, gains_f32;
};
struct NormGradArgs {
    size_t rows, cols;
    const void *r, *y, *gate, *post_gain, *pre_gain, *dz, *dr;
    size_t ldr, ldy, ldgate, lddz, lddr;
    void *dx, *dy, *dgate;
    size_t lddx, lddy, lddgate;
    float* partial;        // [blocks][3][cols]: sums for the gains and the gate over the rows of each block
    float scale, eps;
    int gate_kind;
    bool post_norm, pre_norm, gains_f32, want_pre, want_post, want_gate;
};

// Sums of K values over the threads of a row (blockDim.x of them, whole warps), for every thread.  `buf` holds 32 * K floats
// of the row's own; a call may follow another on the same buffer only after a barrier.
template <int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* buf) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    const unsigned warps = blockDim.x >> 5;
    if (warps == 1) return;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) buf[k * 32 + (threadIdx.x >> 5)] = v[k];
    __syncthreads();
    const unsigned lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane < warps ? buf[k * 32 + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}

template <class T, int V>
__device__ __forceinline__ void load_gain(const void* p, bool f32, size_t at, float (&out)[V]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = 1.0f;
    } else if (f32) {
        constexpr int W = V < 4 ? V : 4;
#pragma unroll
        for (int i = 0; i < V; i += W) {
            float w[W];
            load_vec<float, W>(static_cast<const float*>(p) + at + i, w);
#pragma unroll
            for (int j = 0; j < W; ++j) out[i + j] = w[j];
        }
    } else {
        load_vec<T, V>(static_cast<const T*>(p) + at, out);
    }
}

// the gate's values at one place of a row
template <class T, int V>
__device__ __forceinline__ void load_gate(const void* p, int kind, bool gains_f32, size_t ld, size_t row, size_t at, float (&out)[V]) {
    if (kind == ZKB_GATE_ELEMENT) {
        load_vec<T, V>(static_cast<const T*>(p) + row * ld + at, out);
    } else if (kind == ZKB_GATE_CHANNEL) {
        load_gain<T, V>(p, gains_f32, at, out);
    } else {
        const float g = kind == ZKB_GATE_ROW ? to_f32<T>(static_cast<const T*>(p)[row]) : 1.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = g;
    }
}

// Bound by HBM: x and y are read once, r and z written once, and a row stays in registers between its two sums.
// NV vectors of V values to a thread, blockDim.x threads to a row, blockDim.y rows to a block.
template <class T, int V, int NV>
__global__ void __launch_bounds__(1024) block_norm_kernel(const __grid_constant__ NormArgs a) {
    extern __shared__ float sums[];
    float* buf = sums + threadIdx.y * 64;
    const size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
    const bool live = row < a.rows;
    float x[NV][V], y[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
        const bool in = live && at < a.cols;
#pragma unroll
        for (int j = 0; j < V; ++j) x[i][j] = y[i][j] = 0.0f;
        if (in) load_vec<T, V>(static_cast<const T*>(a.x) + row * a.ldx + at, x[i]);
        if (in && a.y) load_vec<T, V>(static_cast<const T*>(a.y) + row * a.ldy + at, y[i]);
    }
    float post_inv = 1.0f;
    if (a.post_norm) {
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += y[i][j] * y[i][j];
        row_sum<1>(s, buf);
        post_inv = rsqrtf(s[0] / (float)a.cols + a.eps);
        if (live && threadIdx.x == 0 && a.post_inv) a.post_inv[row] = post_inv;
    }
    float s[1] = {0.0f};
    if (a.y) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
            if (!live || at >= a.cols) continue;
            float w[V], g[V];
            load_gain<T, V>(a.post_gain, a.gains_f32, at, w);
            load_gate<T, V>(a.gate, a.gate_kind, a.gains_f32, a.ldgate, row, at, g);
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] += a.scale * g[j] * (y[i][j] * post_inv * w[j]);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
        if (a.r && live && at < a.cols) store_vec<T, V>(static_cast<T*>(a.r) + row * a.ldr + at, x[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) s[0] += x[i][j] * x[i][j];
    }
    if (!a.pre_norm) return;
    row_sum<1>(s, buf + 32);
    const float inv = rsqrtf(s[0] / (float)a.cols + a.eps);
    if (!live) return;
    if (threadIdx.x == 0 && a.pre_inv) a.pre_inv[row] = inv;
    if (!a.z) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
        if (at >= a.cols) continue;
        float w[V];
        load_gain<T, V>(a.pre_gain, a.gains_f32, at, w);
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] *= x[i][j] * inv;
        store_vec<T, V>(static_cast<T*>(a.z) + row * a.ldz + at, w);
    }
}

// The gradients.  With p = dz * w_pre, the gradient of r is d = dr + inv (p - r inv^2 mean(p r)); that of the branch before
// its norm follows from dn = a * gate * d in the same way.  Each block takes rows blockIdx.x, blockIdx.x + gridDim.x, ... and keeps
// its share of the gains' and the gate's sums over rows in registers; norm_reduce_kernel adds the blocks' shares in their order, so
// that a result does not depend on timing.
template <class T, int V, int NV, int kThreads>
__global__ void __launch_bounds__(kThreads) block_norm_backward_kernel(const __grid_constant__ NormGradArgs a) {
    __shared__ float sums[5 * 32];
    float acc_pre[NV][V], acc_post[NV][V], acc_gate[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc_pre[i][j] = acc_post[i][j] = acc_gate[i][j] = 0.0f;
    const float count = (float)a.cols;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float r[NV][V], y[NV][V], dz[NV][V];
        float s[3] = {0.0f, 0.0f, 0.0f};   // r^2, p r, y^2
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) r[i][j] = y[i][j] = dz[i][j] = 0.0f;
            if (at >= a.cols) continue;
            if (a.pre_norm) {
                load_vec<T, V>(static_cast<const T*>(a.r) + row * a.ldr + at, r[i]);
                load_vec<T, V>(static_cast<const T*>(a.dz) + row * a.lddz + at, dz[i]);
            }
            if (a.y) load_vec<T, V>(static_cast<const T*>(a.y) + row * a.ldy + at, y[i]);
            float w[V];
            load_gain<T, V>(a.pre_gain, a.gains_f32, at, w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s[0] += r[i][j] * r[i][j];
                s[1] += dz[i][j] * w[j] * r[i][j];
                s[2] += y[i][j] * y[i][j];
            }
        }
        row_sum<3>(s, sums);
        const float inv = a.pre_norm ? rsqrtf(s[0] / count + a.eps) : 0.0f;
        const float back = inv * inv * s[1] / count;
        const float post_inv = a.post_norm ? rsqrtf(s[2] / count + a.eps) : 1.0f;
        float q[2] = {0.0f, 0.0f};          // dn w_post y, d n
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
            if (at >= a.cols) continue;
            float w[V], d[V];
            load_gain<T, V>(a.pre_gain, a.gains_f32, at, w);
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = 0.0f;
            if (a.dr) load_vec<T, V>(static_cast<const T*>(a.dr) + row * a.lddr + at, d);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                acc_pre[i][j] += dz[i][j] * (r[i][j] * inv);
                d[j] += inv * (dz[i][j] * w[j] - r[i][j] * back);
                r[i][j] = d[j];             // from here on: the gradient of r
            }
            if (a.dx) store_vec<T, V>(static_cast<T*>(a.dx) + row * a.lddx + at, d);
            if (!a.y) continue;
            float wp[V], g[V], dg[V];
            load_gain<T, V>(a.post_gain, a.gains_f32, at, wp);
            load_gate<T, V>(a.gate, a.gate_kind, a.gains_f32, a.ldgate, row, at, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float yn = y[i][j] * post_inv;
                const float dn = a.scale * g[j] * d[j];
                q[0] += dn * wp[j] * y[i][j];
                q[1] += d[j] * (yn * wp[j]);
                acc_post[i][j] += dn * yn;
                dg[j] = a.scale * d[j] * (yn * wp[j]);
                acc_gate[i][j] += dg[j];
                dz[i][j] = dn * wp[j];      // from here on: the gradient of the normed branch times its gain
            }
            if (a.want_gate && a.gate_kind == ZKB_GATE_ELEMENT) store_vec<T, V>(static_cast<T*>(a.dgate) + row * a.lddgate + at, dg);
        }
        if (!a.y) { __syncthreads(); continue; }
        row_sum<2>(q, sums + 96);
        if (a.want_gate && a.gate_kind == ZKB_GATE_ROW && threadIdx.x == 0) static_cast<T*>(a.dgate)[row] = from_f32<T>(a.scale * q[1]);
        const float post_back = a.post_norm ? post_inv * post_inv * q[0] / count : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
            if (!a.dy || at >= a.cols) continue;
            float dy[V];
#pragma unroll
            for (int j = 0; j < V; ++j) dy[j] = post_inv * (dz[i][j] - y[i][j] * post_back);
            store_vec<T, V>(static_cast<T*>(a.dy) + row * a.lddy + at, dy);
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (size_t)blockIdx.x * 3 * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
        if (at >= a.cols) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (a.want_pre) out[at + j] = acc_pre[i][j];
            if (a.want_post) out[a.cols + at + j] = acc_post[i][j];
            if (a.want_gate) out[2 * a.cols + at + j] = acc_gate[i][j];
        }
    }
}

// Adds the blocks' shares: blockIdx.y says of which vector (null: not asked for).
template <class T>
__global__ void norm_reduce_kernel(const float* __restrict__ partial, unsigned blocks, size_t cols, void* d0, void* d1, void* d2, bool f32) {
    void* out = blockIdx.y == 0 ? d0 : blockIdx.y == 1 ? d1 : d2;
    const size_t c = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (!out || c >= cols) return;
    float s = 0.0f;
    for (unsigned b = 0; b < blocks; ++b) s += partial[((size_t)b * 3 + blockIdx.y) * cols + c];
    if (f32) static_cast<float*>(out)[c] = s;
    else static_cast<T*>(out)[c] = from_f32<T>(s);
}

// threads to a row for `per` values a thread, whole warps
unsigned row_threads(size_t cols, unsigned per) { return std::max(32u, div_up(div_up(cols, per), 32) * 32); }

template <class T>
int norm_launch(const NormArgs& a, bool wide, cudaStream_t s) {
    constexpr int W = kWide<T>;
    // 8 values to a thread, 16 where a row would need more than 1024 threads
    const unsigned per = wide ? (a.cols > 8192 ? 16 : 8) : (a.cols > 4096 ? 16 : 4);
    const unsigned tx = row_threads(a.cols, per), ty = std::max(1u, 128 / tx);
    const auto block_norm = wide ? (per == 16 ? block_norm_kernel<T, W, 16 / W> : block_norm_kernel<T, W, 8 / W>)
                                 : (per == 16 ? block_norm_kernel<T, 1, 16> : block_norm_kernel<T, 1, 4>);
    ZKB_LAUNCH(block_norm, div_up(a.rows, ty), dim3(tx, ty), ty * 64 * sizeof(float), s, a);
    return ZKB_OK;
}

template <class T>
int norm_backward_launch(NormGradArgs a, bool wide, void* dpost, void* dpre, cudaStream_t s) {
    constexpr int W = kWide<T>;
    const unsigned per = wide ? (a.cols > 2048 ? 16 : 8) : (a.cols > 2048 ? 16 : 4);
    const unsigned tx = row_threads(a.cols, per);
    const auto block_norm_backward =
        tx > 512 ? (wide ? block_norm_backward_kernel<T, W, 16 / W, 1024> : block_norm_backward_kernel<T, 1, 16, 1024>)
                 : wide ? (per == 16 ? block_norm_backward_kernel<T, W, 16 / W, 512> : block_norm_backward_kernel<T, W, 8 / W, 512>)
                        : (per == 16 ? block_norm_backward_kernel<T, 1, 16, 512> : block_norm_backward_kernel<T, 1, 4, 512>);
    int resident = 1;
    ZKB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, block_norm_backward, tx, 0));
    const unsigned blocks = (unsigned)std::min<size_t>(a.rows, (size_t)std::max(resident, 1) * sm_count());
    Scratch scratch(s);
    const bool channel = a.want_gate && a.gate_kind == ZKB_GATE_CHANNEL;
    if (a.want_pre || a.want_post || channel) {
        a.partial = scratch.get_n<float>((size_t)blocks * 3 * a.cols);
        if (!a.partial) return ZKB_ERR_CUDA;
    }
    ZKB_LAUNCH(block_norm_backward, blocks, tx, 0, s, a);
    if (a.partial) {
        const auto norm_reduce = norm_reduce_kernel<T>;
        ZKB_LAUNCH(norm_reduce, dim3(div_up(a.cols, 128), 3), 128, 0, s, a.partial, blocks, a.cols, dpre, dpost, channel ? a.dgate : nullptr,
                   a.gains_f32);
    }
    return ZKB_OK;
}

// what both directions check
int check_common(const char* who, int dtype, int gains_dtype, size_t rows, size_t cols, const void* y, int post_norm, const void* post_gain, int gate_kind,
                 const void* gate, float eps, float scale) {
    const std::string w(who);
    if (!known_type(dtype)) return fail(ZKB_ERR_ARG, w + ": unknown type");
    if (gains_dtype != dtype && gains_dtype != ZKB_F32) return fail(ZKB_ERR_ARG, w + ": gains are of the tensors' type or f32");
    if (cols > kMaxCols) return fail(ZKB_ERR_LIMIT, w + ": rows of more than 16384 values");
    if (rows > 0x7fffffffull) return fail(ZKB_ERR_LIMIT, w + ": 2^31 rows or more");
    if (!(eps > 0.0f) || !std::isfinite(eps)) return fail(ZKB_ERR_ARG, w + ": eps has to be positive and finite");
    if (!std::isfinite(scale)) return fail(ZKB_ERR_ARG, w + ": residual scale is not finite");
    if (gate_kind < ZKB_GATE_NONE || gate_kind > ZKB_GATE_ELEMENT) return fail(ZKB_ERR_ARG, w + ": unknown kind of gate");
    if ((gate_kind != ZKB_GATE_NONE) != (gate != nullptr)) return fail(ZKB_ERR_ARG, w + ": gate and its kind do not agree");
    if (!y && (post_norm || gate || post_gain)) return fail(ZKB_ERR_ARG, w + ": a norm, gain or gate without a branch");
    if (post_gain && !post_norm) return fail(ZKB_ERR_ARG, w + ": a gain without its norm");
    return ZKB_OK;
}
struct Matrix { const void* p; size_t ld; const char* name; };
int check_matrix(const char* who, const Matrix& m, int dtype, size_t rows, size_t cols, bool* wide) {
    if (!m.p) return ZKB_OK;
    const std::string w = std::string(who) + ": " + m.name;
    if (m.ld < cols && rows > 1) return fail(ZKB_ERR_DIM, w + ": row stride below the row's length");
    ZKB_TRY(check_device(m.p, type_size(dtype), w.c_str()));
    if (!aligned_to(m.p, 16) || (m.ld * type_size(dtype)) % 16) *wide = false;
    return ZKB_OK;
}
int check_vector(const char* who, const void* p, const char* name, int dtype, bool* wide) {
    if (!p) return ZKB_OK;
    ZKB_TRY(check_device(p, type_size(dtype), (std::string(who) + ": " + name).c_str()));
    if (!aligned_to(p, 16)) *wide = false;
    return ZKB_OK;
}

}  // namespace
}  // namespace zkb

using namespace zkb;

extern "C" {

int zkb_block_norm(int dtype, int gains_dtype, size_t rows, size_t cols, const void* d_x, size_t ldx, const void* d_y, size_t ldy, int post_norm,
                   const void* d_post_gain, int gate_kind, const void* d_gate, size_t ldgate, float residual_scale, int pre_norm,
                   const void* d_pre_gain, float eps, void* d_r, size_t ldr, void* d_z, size_t ldz, float* d_post_inv, float* d_pre_inv, void* stream) {
    ZKB_API_RANGE();
    const char* who = "zkb_block_norm";
    ZKB_TRY(check_common(who, dtype, gains_dtype, rows, cols, d_y, post_norm, d_post_gain, gate_kind, d_gate, eps, residual_scale));
    if (!pre_norm && (d_z || d_pre_gain || d_pre_inv)) return fail(ZKB_ERR_ARG, "zkb_block_norm: z, its gain or its statistics without the norm");
    if (!post_norm && d_post_inv) return fail(ZKB_ERR_ARG, "zkb_block_norm: statistics of the branch without its norm");
    if (!rows || !cols) return ZKB_OK;
    if (!d_x) return fail(ZKB_ERR_ARG, "zkb_block_norm: no x");
    bool wide = cols % (16 / type_size(dtype)) == 0;
    const size_t gate_ld = gate_kind == ZKB_GATE_ELEMENT ? ldgate : 0;
    for (const Matrix& m : {Matrix{d_x, ldx, "x"}, Matrix{d_y, ldy, "y"}, Matrix{d_r, ldr, "r"}, Matrix{d_z, ldz, "z"},
                            Matrix{gate_kind == ZKB_GATE_ELEMENT ? d_gate : nullptr, gate_ld, "gate"}})
        ZKB_TRY(check_matrix(who, m, dtype, rows, cols, &wide));
    ZKB_TRY(check_vector(who, d_post_gain, "post_gain", gains_dtype, &wide));
    ZKB_TRY(check_vector(who, d_pre_gain, "pre_gain", gains_dtype, &wide));
    if (gate_kind == ZKB_GATE_CHANNEL) ZKB_TRY(check_vector(who, d_gate, "gate", gains_dtype, &wide));
    bool any = true;
    if (gate_kind == ZKB_GATE_ROW) ZKB_TRY(check_vector(who, d_gate, "gate", dtype, &any));
    ZKB_TRY(check_vector(who, d_post_inv, "post_inv", ZKB_F32, &any));
    ZKB_TRY(check_vector(who, d_pre_inv, "pre_inv", ZKB_F32, &any));
    const NormArgs a = {rows, cols, d_x, d_y, d_gate, d_post_gain, d_pre_gain, ldx, ldy, gate_ld, d_r, d_z, ldr, ldz, d_post_inv, d_pre_inv,
                        residual_scale, eps, gate_kind, post_norm != 0, pre_norm != 0, gains_dtype == ZKB_F32};
    const cudaStream_t s = as_stream(stream);
    if (dtype == ZKB_F32) return norm_launch<float>(a, wide, s);
    if (dtype == ZKB_F16) return norm_launch<__half>(a, wide, s);
    return norm_launch<bf16>(a, wide, s);
}

int zkb_block_norm_backward(int dtype, int gains_dtype, size_t rows, size_t cols, const void* d_r, size_t ldr, const void* d_y, size_t ldy, int post_norm,
                            const void* d_post_gain, int gate_kind, const void* d_gate, size_t ldgate, float residual_scale, int pre_norm,
                            const void* d_pre_gain, float eps, const void* d_dz, size_t lddz, const void* d_dr, size_t lddr, void* d_dx, size_t lddx,
                            void* d_dy, size_t lddy, void* d_dgate, size_t lddgate, void* d_dpost_gain, void* d_dpre_gain, void* stream) {
    ZKB_API_RANGE();
    const char* who = "zkb_block_norm_backward";
    ZKB_TRY(check_common(who, dtype, gains_dtype, rows, cols, d_y, post_norm, d_post_gain, gate_kind, d_gate, eps, residual_scale));
    if (!pre_norm && (d_dz || d_pre_gain || d_dpre_gain)) return fail(ZKB_ERR_ARG, "zkb_block_norm_backward: z's gradient or gain without the norm");
    if (!d_y && (d_dy || d_dpost_gain || d_dgate)) return fail(ZKB_ERR_ARG, "zkb_block_norm_backward: a branch's gradient without the branch");
    if (!post_norm && d_dpost_gain) return fail(ZKB_ERR_ARG, "zkb_block_norm_backward: a gain's gradient without its norm");
    if (gate_kind == ZKB_GATE_NONE && d_dgate) return fail(ZKB_ERR_ARG, "zkb_block_norm_backward: a gate's gradient without the gate");
    if (!cols) return ZKB_OK;
    const size_t gb = type_size(gains_dtype);
    const cudaStream_t s = as_stream(stream);
    bool wide = cols % (16 / type_size(dtype)) == 0, any = true;
    ZKB_TRY(check_vector(who, d_dpost_gain, "dpost_gain", gains_dtype, &any));
    ZKB_TRY(check_vector(who, d_dpre_gain, "dpre_gain", gains_dtype, &any));
    if (!rows) {   // a sum over no rows
        if (d_dpost_gain) ZKB_CUDA(cudaMemsetAsync(d_dpost_gain, 0, cols * gb, s));
        if (d_dpre_gain) ZKB_CUDA(cudaMemsetAsync(d_dpre_gain, 0, cols * gb, s));
        if (d_dgate && gate_kind == ZKB_GATE_CHANNEL) {
            ZKB_TRY(check_vector(who, d_dgate, "dgate", gains_dtype, &any));
            ZKB_CUDA(cudaMemsetAsync(d_dgate, 0, cols * gb, s));
        }
        return ZKB_OK;
    }
    if (pre_norm && (!d_r || !d_dz)) return fail(ZKB_ERR_ARG, "zkb_block_norm_backward: no r or no gradient of z");
    const bool element = gate_kind == ZKB_GATE_ELEMENT;
    const size_t gate_ld = element ? ldgate : 0;
    for (const Matrix& m : {Matrix{d_r, ldr, "r"}, Matrix{d_y, ldy, "y"}, Matrix{d_dz, lddz, "dz"}, Matrix{d_dr, lddr, "dr"}, Matrix{d_dx, lddx, "dx"},
                            Matrix{d_dy, lddy, "dy"}, Matrix{element ? d_gate : nullptr, gate_ld, "gate"}, Matrix{element ? d_dgate : nullptr, lddgate, "dgate"}})
        ZKB_TRY(check_matrix(who, m, dtype, rows, cols, &wide));
    ZKB_TRY(check_vector(who, d_post_gain, "post_gain", gains_dtype, &wide));
    ZKB_TRY(check_vector(who, d_pre_gain, "pre_gain", gains_dtype, &wide));
    if (gate_kind == ZKB_GATE_CHANNEL) {
        ZKB_TRY(check_vector(who, d_gate, "gate", gains_dtype, &wide));
        ZKB_TRY(check_vector(who, d_dgate, "dgate", gains_dtype, &any));
    } else if (gate_kind == ZKB_GATE_ROW) {
        ZKB_TRY(check_vector(who, d_gate, "gate", dtype, &any));
        ZKB_TRY(check_vector(who, d_dgate, "dgate", dtype, &any));
    }
    NormGradArgs a = {rows, cols, d_r, d_y, d_gate, d_post_gain, d_pre_gain, d_dz, d_dr, ldr, ldy, gate_ld, lddz, lddr, d_dx, d_dy, d_dgate, lddx, lddy, lddgate,
                      nullptr, residual_scale, eps, gate_kind, post_norm != 0, pre_norm != 0, gains_dtype == ZKB_F32, d_dpre_gain != nullptr,
                      d_dpost_gain != nullptr, d_dgate != nullptr};
    if (dtype == ZKB_F32) return norm_backward_launch<float>(a, wide, d_dpost_gain, d_dpre_gain, s);
    if (dtype == ZKB_F16) return norm_backward_launch<__half>(a, wide, d_dpost_gain, d_dpre_gain, s);
    return norm_backward_launch<bf16>(a, wide, d_dpost_gain, d_dpre_gain, s);
}

}  // extern "C"
