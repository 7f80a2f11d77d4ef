// The norms after one branch of a layer and before the next, with the branch's gate, residual scale and addition between them.
//
//     n = y / sqrt(mean y^2 + eps) * w_post      (or y, without the norm after the branch)
//     r = x + a * gate * n
//     z = r / sqrt(mean r^2 + eps) * w_pre
//
// and the gradients of x, y, the gate and both gains.  Sums are in 32 bits; z is formed from r before r is rounded.
#include <algorithm>

#include "tensorcore.cuh"

namespace zkb {
namespace {

constexpr size_t kMaxCols = 16384;

// Rows of a matrix that a kernel reads: null for one that the call lacks.
struct Source {
    const char* p;
    size_t ld;       // in bytes
    unsigned at;     // its place in a slot, bytes
};

struct NormArgs {
    size_t rows, cols;
    Source src[3];         // x, y, gate values
    const void *gate, *post_gain, *pre_gain;
    void *r, *z;
    size_t ldr, ldz;
    float *post_inv, *pre_inv;
    float scale, eps;
    int gate_kind;
    bool post_norm, pre_norm, gains_f32;
    unsigned slots, slot_bytes;
    int* flag;
};
struct NormGradArgs {
    size_t rows, cols;
    Source src[5];         // r, dz, y, dr, gate values
    const void *gate, *post_gain, *pre_gain;
    void *dx, *dy, *dgate;
    size_t lddx, lddy, lddgate;
    float* partial;        // [blocks][2][cols]: each block's sums over its rows
    float scale, eps;
    int gate_kind;
    bool post_norm, pre_norm, gains_f32, want_gate;
    unsigned slots, slot_bytes;
    int* flag;
};

// Rows on their way: a block's next rows are copied into a ring of slots in shared memory while it works on the present one, up to N
// matrices to a slot.  A row may begin at any element: the copy takes the whole 16-byte granules that it lies in.  The first and the
// last of these hold at least one byte of the row each, so that nothing beyond the row's own pages is read.
__host__ __device__ __forceinline__ unsigned slot_row_bytes(size_t cols, size_t es) { return (unsigned)(cols * es + 30) / 16 * 16; }
template <class T, int N>
struct RowRing {
    const Source* src;
    char* slots;
    uint32_t bars, row_bytes, slot_bytes;
    unsigned n_slots;
    tc::Watch watch;

    __device__ __forceinline__ RowRing(const Source* source, size_t cols, unsigned count, unsigned bytes, char* memory, int* flag)
        : src(source), slots(memory + 16 * 8), bars(tc::smem_address(memory)), row_bytes((uint32_t)(cols * sizeof(T))),
          slot_bytes(bytes), n_slots(count), watch{reinterpret_cast<volatile int*>(memory + 15 * 8), flag} {
        if (threadIdx.x == 0) {
            for (unsigned i = 0; i < n_slots; ++i) tc::barrier_init(bars + 8 * i, 1);
            *watch.dead = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    // one thread: the copies of a row into a slot
    __device__ __forceinline__ void fetch(size_t row, unsigned slot) const {
        uint32_t bytes = 0;
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (src[k].p) {
                const unsigned long long at = reinterpret_cast<unsigned long long>(src[k].p) + row * src[k].ld;
                bytes += (uint32_t)(((at + row_bytes + 15) & ~15ull) - (at & ~15ull));
            }
        if (!bytes) {
            tc::barrier_arrive(bars + 8 * slot);
            return;
        }
        tc::barrier_expect(bars + 8 * slot, bytes);
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (src[k].p) {
                const unsigned long long at = reinterpret_cast<unsigned long long>(src[k].p) + row * src[k].ld;
                tc::load_bytes(tc::smem_address(slots) + slot * slot_bytes + src[k].at, at & ~15ull, (uint32_t)(((at + row_bytes + 15) & ~15ull) - (at & ~15ull)),
                               bars + 8 * slot);
            }
    }
    __device__ __forceinline__ void wait(unsigned slot, uint32_t parity) const { tc::barrier_wait(bars + 8 * slot, parity, watch); }
    __device__ __forceinline__ const T* row_of(int k, size_t row, unsigned slot) const {
        const unsigned long long at = reinterpret_cast<unsigned long long>(src[k].p) + row * src[k].ld;
        return reinterpret_cast<const T*>(slots + slot * slot_bytes + src[k].at + (at & 15));
    }
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

// the gate's values at one place of a row; `values` is an ELEMENT gate's row, `row_gate` a ROW gate's value
template <class T, int V>
__device__ __forceinline__ void load_gate(const void* p, const T* values, int kind, bool gains_f32, float row_gate, size_t at, float (&out)[V]) {
    if (kind == ZKB_GATE_ELEMENT) {
        load_vec<T, V>(values + at, out);
    } else if (kind == ZKB_GATE_CHANNEL) {
        load_gain<T, V>(p, gains_f32, at, out);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = row_gate;
    }
}

// Bound by HBM: x and y are read once, r and z written once.  Each block takes rows blockIdx.x, blockIdx.x + gridDim.x, ...; with
// kRing their values come through the ring, else straight from global memory (rows too long for two slots, or few rows, where
// nothing could be fetched ahead).  NV vectors of V values to a thread.
template <class T, int V, int NV, int kThreads, int kBlocks, bool kRing>
__global__ void __launch_bounds__(kThreads, kBlocks) block_norm_kernel(const __grid_constant__ NormArgs a) {
    extern __shared__ __align__(16) char memory[];
    __shared__ float sums[2 * 32];
    grid_release();
    const RowRing<T, 3> ring(a.src, kRing ? a.cols : 0, kRing ? a.slots : 0, kRing ? a.slot_bytes : 0, memory, a.flag);
    grid_wait();
    if (kRing && threadIdx.x == 0)
        for (unsigned i = 0; i < a.slots && blockIdx.x + (size_t)i * gridDim.x < a.rows; ++i) ring.fetch(blockIdx.x + (size_t)i * gridDim.x, i);
    const bool branch = a.src[1].p != nullptr;
    unsigned slot = 0;
    uint32_t phase = 0;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (kRing) ring.wait(slot, phase);
        const T* from[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) from[k] = kRing ? ring.row_of(k, row, slot) : reinterpret_cast<const T*>(a.src[k].p + row * a.src[k].ld);
        float x[NV][V], y[NV][V];
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = y[i][j] = 0.0f;
            if (at >= a.cols) continue;
            load_vec<T, V>(from[0] + at, x[i]);
            if (!branch) continue;
            load_vec<T, V>(from[1] + at, y[i]);
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += y[i][j] * y[i][j];
        }
        float post_inv = 1.0f;
        if (a.post_norm) {
            row_sum<1>(s, sums);
            post_inv = rsqrtf(s[0] / (float)a.cols + a.eps);
            if (threadIdx.x == 0 && a.post_inv) a.post_inv[row] = post_inv;
        }
        if (branch) {
            const float row_gate = a.gate_kind == ZKB_GATE_ROW ? to_f32<T>(static_cast<const T*>(a.gate)[row]) : 1.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
                if (at >= a.cols) continue;
                float w[V], g[V];
                load_gain<T, V>(a.post_gain, a.gains_f32, at, w);
                load_gate<T, V>(a.gate, from[2], a.gate_kind, a.gains_f32, row_gate, at, g);
#pragma unroll
                for (int j = 0; j < V; ++j) x[i][j] += a.scale * g[j] * (y[i][j] * post_inv * w[j]);
            }
        }
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
            if (a.r && at < a.cols) store_vec<T, V>(static_cast<T*>(a.r) + row * a.ldr + at, x[i]);
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += x[i][j] * x[i][j];
        }
        row_sum<1>(s, sums + 32);
        __syncthreads();      // one warp alone passes no barrier in row_sum; every thread is done with this row's slot
        if (kRing) {
            const size_t next = row + (size_t)a.slots * gridDim.x;
            if (threadIdx.x == 0 && next < a.rows) ring.fetch(next, slot);
            if (++slot == a.slots) { slot = 0; phase ^= 1; }
        }
        if (!a.pre_norm) continue;
        const float inv = rsqrtf(s[0] / (float)a.cols + a.eps);
        if (threadIdx.x == 0 && a.pre_inv) a.pre_inv[row] = inv;
        if (!a.z) continue;
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
}

// The gradients.  With p = dz * w_pre, the gradient of r is d = dr + inv (p - r inv^2 mean(p r)); that of the branch before
// its norm follows from a * gate * d * w_post in the same way.  Two sums over rows serve all three vectors: dz r inv gives the
// gain before the next branch, and S = d yn (times the gate where that is not the same for all rows) both the other gain,
// a gate S, and a CHANNEL gate, a w_post S.  Each block keeps its rows' share of them in registers; norm_reduce_kernel adds the
// shares in the order of the blocks, so that a result does not depend on timing.
template <class T, int V, int NV, int kThreads, int kBlocks, bool kRing>
__global__ void __launch_bounds__(kThreads, kBlocks) block_norm_backward_kernel(const __grid_constant__ NormGradArgs a) {
    extern __shared__ __align__(16) char memory[];
    __shared__ float sums[5 * 32];
    grid_release();
    const RowRing<T, 5> ring(a.src, kRing ? a.cols : 0, kRing ? a.slots : 0, kRing ? a.slot_bytes : 0, memory, a.flag);
    grid_wait();
    if (kRing && threadIdx.x == 0)
        for (unsigned i = 0; i < a.slots && blockIdx.x + (size_t)i * gridDim.x < a.rows; ++i) ring.fetch(blockIdx.x + (size_t)i * gridDim.x, i);
    const bool branch = a.src[2].p != nullptr, more = a.src[3].p != nullptr;
    const float count = (float)a.cols;
    float acc_pre[NV][V], acc_post[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc_pre[i][j] = acc_post[i][j] = 0.0f;
    unsigned slot = 0;
    uint32_t phase = 0;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (kRing) ring.wait(slot, phase);
        const T* from[5];
#pragma unroll
        for (int k = 0; k < 5; ++k) from[k] = kRing ? ring.row_of(k, row, slot) : reinterpret_cast<const T*>(a.src[k].p + row * a.src[k].ld);
        float s[3] = {0.0f, 0.0f, 0.0f};   // r^2, p r, y^2
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
            if (at >= a.cols) continue;
            if (a.pre_norm) {
                float r[V], dz[V], w[V];
                load_vec<T, V>(from[0] + at, r);
                load_vec<T, V>(from[1] + at, dz);
                load_gain<T, V>(a.pre_gain, a.gains_f32, at, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s[0] += r[j] * r[j];
                    s[1] += dz[j] * w[j] * r[j];
                }
            }
            if (a.post_norm) {
                float y[V];
                load_vec<T, V>(from[2] + at, y);
#pragma unroll
                for (int j = 0; j < V; ++j) s[2] += y[j] * y[j];
            }
        }
        row_sum<3>(s, sums);
        const float inv = a.pre_norm ? rsqrtf(s[0] / count + a.eps) : 0.0f;
        const float back = inv * inv * s[1] / count;
        const float post_inv = a.post_norm ? rsqrtf(s[2] / count + a.eps) : 1.0f;
        const float row_gate = a.gate_kind == ZKB_GATE_ROW ? to_f32<T>(static_cast<const T*>(a.gate)[row]) : 1.0f;
        const bool by_row = a.gate_kind == ZKB_GATE_ROW || a.gate_kind == ZKB_GATE_ELEMENT;
        float q[2] = {0.0f, 0.0f};          // gate w_post d y, w_post d y
        float d[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
            if (at >= a.cols) continue;
#pragma unroll
            for (int j = 0; j < V; ++j) d[i][j] = 0.0f;
            if (more) load_vec<T, V>(from[3] + at, d[i]);
            if (a.pre_norm) {
                float r[V], dz[V], w[V];
                load_vec<T, V>(from[0] + at, r);
                load_vec<T, V>(from[1] + at, dz);
                load_gain<T, V>(a.pre_gain, a.gains_f32, at, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    acc_pre[i][j] += dz[j] * (r[j] * inv);
                    d[i][j] += inv * (dz[j] * w[j] - r[j] * back);
                }
            }
            if (a.dx) store_vec<T, V>(static_cast<T*>(a.dx) + row * a.lddx + at, d[i]);
            if (!branch) continue;
            float y[V], wp[V], g[V];
            load_vec<T, V>(from[2] + at, y);
            load_gain<T, V>(a.post_gain, a.gains_f32, at, wp);
            load_gate<T, V>(a.gate, from[4], a.gate_kind, a.gains_f32, row_gate, at, g);
            if (a.gate_kind == ZKB_GATE_ELEMENT && a.want_gate) {
                float dg[V];
#pragma unroll
                for (int j = 0; j < V; ++j) dg[j] = a.scale * d[i][j] * (y[j] * post_inv * wp[j]);
                store_vec<T, V>(static_cast<T*>(a.dgate) + row * a.lddgate + at, dg);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float dy = d[i][j] * y[j];
                acc_post[i][j] += by_row ? g[j] * (dy * post_inv) : dy * post_inv;
                q[0] += g[j] * wp[j] * dy;
                q[1] += wp[j] * dy;
                d[i][j] *= g[j] * wp[j];    // from here on: the gradient of the normed branch times its gain, less the scale
            }
        }
        row_sum<2>(q, sums + 96);
        if (branch) {
            if (a.want_gate && a.gate_kind == ZKB_GATE_ROW && threadIdx.x == 0)
                static_cast<T*>(a.dgate)[row] = from_f32<T>(a.scale * post_inv * q[1]);
            const float post_back = a.post_norm ? post_inv * post_inv * q[0] / count : 0.0f;
            if (a.dy) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
                    if (at >= a.cols) continue;
                    float y[V];
                    load_vec<T, V>(from[2] + at, y);
#pragma unroll
                    for (int j = 0; j < V; ++j) y[j] = a.scale * post_inv * (d[i][j] - y[j] * post_back);
                    store_vec<T, V>(static_cast<T*>(a.dy) + row * a.lddy + at, y);
                }
            }
        }
        __syncthreads();      // every thread is done with this row's slot and sums
        if (kRing) {
            const size_t next = row + (size_t)a.slots * gridDim.x;
            if (threadIdx.x == 0 && next < a.rows) ring.fetch(next, slot);
            if (++slot == a.slots) { slot = 0; phase ^= 1; }
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (size_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const size_t at = ((size_t)i * blockDim.x + threadIdx.x) * V;
        if (at >= a.cols) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            out[at + j] = acc_pre[i][j];
            out[a.cols + at + j] = acc_post[i][j];
        }
    }
}

// Adds the blocks' shares of 32 columns (8 groups of blocks side by side, then the groups in order) and forms the vectors from the two sums.
struct NormReduceArgs {
    const float* partial;
    unsigned blocks;
    size_t cols;
    void *dpre, *dpost, *dgate;         // null: not asked for
    const void *gate, *post_gain;       // a CHANNEL gate and the gain, or null for ones
    float scale;
    bool gains_f32;
};
template <class T>
__global__ void __launch_bounds__(256) norm_reduce_kernel(const __grid_constant__ NormReduceArgs a) {
    __shared__ float part[8][33];
    grid_release();
    grid_wait();
    const unsigned lane = threadIdx.x & 31, group = threadIdx.x >> 5;
    const size_t c = (size_t)blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < a.cols)
        for (unsigned b = group; b < a.blocks; b += 8) s += a.partial[((size_t)b * 2 + blockIdx.y) * a.cols + c];
    part[group][lane] = s;
    __syncthreads();
    if (group || c >= a.cols) return;
    for (int k = 1; k < 8; ++k) s += part[k][lane];
    auto put = [&](void* out, float v) {
        if (!out) return;
        if (a.gains_f32) static_cast<float*>(out)[c] = v;
        else static_cast<T*>(out)[c] = from_f32<T>(v);
    };
    if (blockIdx.y == 0) {
        put(a.dpre, s);
    } else {
        float g[1], w[1];
        load_gain<T, 1>(a.gate, a.gains_f32, c, g);
        load_gain<T, 1>(a.post_gain, a.gains_f32, c, w);
        put(a.dpost, a.scale * g[0] * s);
        put(a.dgate, a.scale * w[0] * s);
    }
}

// threads to a row for `per` values a thread, whole warps
unsigned row_threads(size_t cols, unsigned per) { return std::max(32u, div_up(div_up(cols, per), 32) * 32); }

constexpr size_t kRingHead = 16 * 8;
// The grid of a kernel over rows, and its ring: as many blocks as are resident, each with as many slots as fit.  Without a second
// row to a block, or room for two slots, there is no ring (slots = 0).
template <class Kernel>
int plan_rows(Kernel ringed, Kernel direct, unsigned threads, Source* src, int matrices, size_t rows, size_t row_bytes, Kernel* kernel, unsigned* blocks,
              unsigned* slots, unsigned* slot_bytes, size_t* smem) {
    int resident = 0;
    ZKB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, ringed, threads, 0));
    resident = std::max(1, resident);
    size_t slot = 0;
    for (int k = 0; k < matrices; ++k) {
        src[k].at = (unsigned)slot;
        if (src[k].p) slot += row_bytes;
    }
    *slot_bytes = (unsigned)slot;
    slot = std::max<size_t>(slot, 16);
    const size_t room = 220 * 1024;
    while (resident > 1 && (room / resident - 2048 - kRingHead) / slot < 2) --resident;   // 1 KB of each block's share is the system's
    const size_t fit = std::min<size_t>(8, (room / resident - 2048 - kRingHead) / slot);
    if (fit >= 2 && rows > (size_t)resident * sm_count()) {
        *kernel = ringed;
        *slots = (unsigned)fit;
        *smem = kRingHead + fit * slot;
        *blocks = (unsigned)resident * sm_count();
        ZKB_CUDA(cudaFuncSetAttribute(ringed, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)*smem));
        return ZKB_OK;
    }
    ZKB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, direct, threads, kRingHead));
    *kernel = direct;
    *slots = 0;
    *smem = kRingHead;
    *blocks = (unsigned)std::min<size_t>(rows, (size_t)std::max(1, resident) * sm_count());
    return ZKB_OK;
}

template <class T, int V, int NV>
int norm_launch(NormArgs a, cudaStream_t s) {
    const unsigned threads = row_threads(a.cols, V * NV);
    const auto pick = [&](bool ring) {
        return threads > 512 ? (ring ? block_norm_kernel<T, V, NV, 1024, 1, true> : block_norm_kernel<T, V, NV, 1024, 1, false>)
                             : (ring ? block_norm_kernel<T, V, NV, 512, 2, true> : block_norm_kernel<T, V, NV, 512, 2, false>);
    };
    auto kernel = pick(true);
    unsigned blocks;
    size_t smem;
    ZKB_TRY(plan_rows(pick(true), pick(false), threads, a.src, 3, a.rows, slot_row_bytes(a.cols, sizeof(T)), &kernel, &blocks, &a.slots,
                      &a.slot_bytes, &smem));
    return launch_beside("block_norm", kernel, blocks, threads, smem, s, a);
}

template <class T, int V, int NV>
int norm_backward_launch(NormGradArgs a, void* dpost, void* dpre, cudaStream_t s) {
    const unsigned threads = row_threads(a.cols, V * NV);
    const auto pick = [&](bool ring) {
        return threads > 512 ? (ring ? block_norm_backward_kernel<T, V, NV, 1024, 1, true> : block_norm_backward_kernel<T, V, NV, 1024, 1, false>)
               : threads > 320 ? (ring ? block_norm_backward_kernel<T, V, NV, 512, 1, true> : block_norm_backward_kernel<T, V, NV, 512, 1, false>)
                               : (ring ? block_norm_backward_kernel<T, V, NV, 320, 2, true> : block_norm_backward_kernel<T, V, NV, 320, 2, false>);
    };
    auto kernel = pick(true);
    unsigned blocks;
    size_t smem;
    ZKB_TRY(plan_rows(pick(true), pick(false), threads, a.src, 5, a.rows, slot_row_bytes(a.cols, sizeof(T)), &kernel, &blocks, &a.slots,
                      &a.slot_bytes, &smem));
    Scratch scratch(s);
    const bool channel = a.want_gate && a.gate_kind == ZKB_GATE_CHANNEL;
    if (dpre || dpost || channel) {
        a.partial = scratch.get_n<float>((size_t)blocks * 2 * a.cols);
        if (!a.partial) return ZKB_ERR_CUDA;
    }
    ZKB_TRY(launch_beside("block_norm_backward", kernel, blocks, threads, smem, s, a));
    if (!a.partial) return ZKB_OK;
    const NormReduceArgs n = {a.partial, blocks, a.cols, dpre, dpost, channel ? a.dgate : nullptr, a.gate_kind == ZKB_GATE_CHANNEL ? a.gate : nullptr,
                              a.post_gain, a.scale, a.gains_f32};
    return launch_beside("norm_reduce", norm_reduce_kernel<T>, dim3(div_up(a.cols, 32), 2), 256, 0, s, n);
}

// 16 values to a thread: more would not leave two blocks their registers, fewer would make the sums over a row cost more than the row
template <class T>
int norm_dispatch(const NormArgs& a, bool wide, cudaStream_t s) {
    return wide ? norm_launch<T, kWide<T>, 16 / kWide<T>>(a, s) : norm_launch<T, 1, 16>(a, s);
}
template <class T>
int norm_backward_dispatch(const NormGradArgs& a, bool wide, void* dpost, void* dpre, cudaStream_t s) {
    return wide ? norm_backward_launch<T, kWide<T>, 16 / kWide<T>>(a, dpost, dpre, s) : norm_backward_launch<T, 1, 16>(a, dpost, dpre, s);
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
    ZKB_TRY(tc::check_wait_flag(who));
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
    const size_t es = type_size(dtype);
    NormArgs a = {};
    a.rows = rows, a.cols = cols;
    a.src[0] = {static_cast<const char*>(d_x), ldx * es};
    a.src[1] = {static_cast<const char*>(d_y), ldy * es};
    a.src[2] = {gate_kind == ZKB_GATE_ELEMENT ? static_cast<const char*>(d_gate) : nullptr, gate_ld * es};
    a.gate = d_gate, a.post_gain = d_post_gain, a.pre_gain = d_pre_gain;
    a.r = d_r, a.z = d_z, a.ldr = ldr, a.ldz = ldz, a.post_inv = d_post_inv, a.pre_inv = d_pre_inv;
    a.scale = residual_scale, a.eps = eps, a.gate_kind = gate_kind;
    a.post_norm = post_norm != 0, a.pre_norm = pre_norm != 0, a.gains_f32 = gains_dtype == ZKB_F32;
    if (!(a.flag = tc::wait_flag())) return ZKB_ERR_CUDA;
    const cudaStream_t s = as_stream(stream);
    if (dtype == ZKB_F32) return norm_dispatch<float>(a, wide, s);
    if (dtype == ZKB_F16) return norm_dispatch<__half>(a, wide, s);
    return norm_dispatch<bf16>(a, wide, s);
}

int zkb_block_norm_backward(int dtype, int gains_dtype, size_t rows, size_t cols, const void* d_r, size_t ldr, const void* d_y, size_t ldy, int post_norm,
                            const void* d_post_gain, int gate_kind, const void* d_gate, size_t ldgate, float residual_scale, int pre_norm,
                            const void* d_pre_gain, float eps, const void* d_dz, size_t lddz, const void* d_dr, size_t lddr, void* d_dx, size_t lddx,
                            void* d_dy, size_t lddy, void* d_dgate, size_t lddgate, void* d_dpost_gain, void* d_dpre_gain, void* stream) {
    ZKB_API_RANGE();
    const char* who = "zkb_block_norm_backward";
    ZKB_TRY(check_common(who, dtype, gains_dtype, rows, cols, d_y, post_norm, d_post_gain, gate_kind, d_gate, eps, residual_scale));
    ZKB_TRY(tc::check_wait_flag(who));
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
    const size_t es = type_size(dtype);
    NormGradArgs a = {};
    a.rows = rows, a.cols = cols;
    a.src[0] = {pre_norm ? static_cast<const char*>(d_r) : nullptr, ldr * es};
    a.src[1] = {static_cast<const char*>(d_dz), lddz * es};
    a.src[2] = {static_cast<const char*>(d_y), ldy * es};
    a.src[3] = {static_cast<const char*>(d_dr), lddr * es};
    a.src[4] = {element ? static_cast<const char*>(d_gate) : nullptr, gate_ld * es};
    a.gate = d_gate, a.post_gain = d_post_gain, a.pre_gain = d_pre_gain;
    a.dx = d_dx, a.dy = d_dy, a.dgate = d_dgate, a.lddx = lddx, a.lddy = lddy, a.lddgate = lddgate;
    a.scale = residual_scale, a.eps = eps, a.gate_kind = gate_kind;
    a.post_norm = post_norm != 0, a.pre_norm = pre_norm != 0, a.gains_f32 = gains_dtype == ZKB_F32, a.want_gate = d_dgate != nullptr;
    if (!(a.flag = tc::wait_flag())) return ZKB_ERR_CUDA;
    if (dtype == ZKB_F32) return norm_backward_dispatch<float>(a, wide, d_dpost_gain, d_dpre_gain, s);
    if (dtype == ZKB_F16) return norm_backward_dispatch<__half>(a, wide, d_dpost_gain, d_dpre_gain, s);
    return norm_backward_dispatch<bf16>(a, wide, d_dpost_gain, d_dpre_gain, s);
}

}  // extern "C"
