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
    float scale, eps, one_over_cols;
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
    float scale, eps, one_over_cols;
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
    // behind a kernel's last row: if a wait ran out, what is in flight lands before the block ends
    __device__ __forceinline__ void close() const {
        if (*watch.dead) tc::pause();
    }
    __device__ __forceinline__ void wait(unsigned slot, uint32_t parity) const { tc::barrier_wait(bars + 8 * slot, parity, watch); }
    // in shared memory
    template <bool kAligned> __device__ __forceinline__ uint32_t row_of(int k, size_t row, unsigned slot) const {
        if (kAligned) return tc::smem_address(slots) + slot * slot_bytes + src[k].at;
        const unsigned at = (unsigned)reinterpret_cast<unsigned long long>(src[k].p) + (unsigned)row * (unsigned)src[k].ld;
        return tc::smem_address(slots) + slot * slot_bytes + src[k].at + (at & 15);
    }
};

// ---- pairs of 32-bit values: one instruction works on both ---------------------------------------------------------------------
struct Pair { unsigned long long v; };
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ Pair pair(float x) { return pair(x, x); }
__device__ __forceinline__ void split(Pair p, float* lo, float* hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*lo), "=f"(*hi) : "l"(p.v)); }
__device__ __forceinline__ float total(Pair p) {
    float lo, hi;
    split(p, &lo, &hi);
    return lo + hi;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair c;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
    return c;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}

template <class T> __device__ __forceinline__ Pair widen(uint32_t two);
template <> __device__ __forceinline__ Pair widen<bf16>(uint32_t two) { return pair(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u)); }
template <> __device__ __forceinline__ Pair widen<__half>(uint32_t two) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
    return pair(f.x, f.y);
}
template <class T> __device__ __forceinline__ uint32_t narrow(Pair p) {
    float lo, hi;
    split(p, &lo, &hi);
    uint32_t two;
    if constexpr (std::is_same<T, bf16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(two) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(two) : "f"(hi), "f"(lo));
    return two;
}

// A thread's share of a row is kShare / G groups of G values (kShare: 8 or 16).  With alignment a group is the 16 bytes at (g * threads + thread) * G;
// without, its values are `threads` apart, so that a warp's accesses still run together.  Places behind the row's end read as zero.
template <class T, bool kAligned> constexpr int kGroup = kAligned ? kWide<T> : 4;

template <bool kAligned, int G> struct Place {
    unsigned at, step, cols;
    __device__ __forceinline__ Place(int g, unsigned n) : at((g * blockDim.x * G) + (kAligned ? threadIdx.x * G : threadIdx.x)), step(blockDim.x), cols(n) {}
    __device__ __forceinline__ bool any() const { return at < cols; }   // aligned: the whole group or nothing
    __device__ __forceinline__ bool has(int j) const { return kAligned || at + j * step < cols; }
    __device__ __forceinline__ unsigned of(int j) const { return kAligned ? at + j : at + j * step; }
};
// Where a row's values are read from: a slot of the ring, or global memory.
template <class T> struct InSlot {
    uint32_t p;
    __device__ __forceinline__ uint4 wide(unsigned at) const {
        uint4 x;
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(p + at * (uint32_t)sizeof(T)));
        return x;
    }
    __device__ __forceinline__ float one(unsigned at) const {
        if constexpr (sizeof(T) == 4) {
            float x;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(p + at * 4));
            return x;
        } else {
            unsigned short x;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(p + at * 2));
            return to_f32<T>(*reinterpret_cast<const T*>(&x));
        }
    }
};
template <class T> struct InMemory {
    const T* p;
    __device__ __forceinline__ uint4 wide(unsigned at) const { return *reinterpret_cast<const uint4*>(p + at); }
    __device__ __forceinline__ float one(unsigned at) const { return to_f32<T>(p[at]); }
};
template <class T, bool kAligned, int G, class From>
__device__ __forceinline__ void load_group(const From& from, const Place<kAligned, G>& at, Pair (&out)[G / 2]) {
    if constexpr (kAligned && sizeof(T) == 2) {
        const uint4 x = from.wide(at.at);
        out[0] = widen<T>(x.x), out[1] = widen<T>(x.y), out[2] = widen<T>(x.z), out[3] = widen<T>(x.w);
    } else if constexpr (kAligned) {
        const uint4 x = from.wide(at.at);
        out[0] = pair(__uint_as_float(x.x), __uint_as_float(x.y)), out[1] = pair(__uint_as_float(x.z), __uint_as_float(x.w));
    } else {
#pragma unroll
        for (int j = 0; j < G; j += 2) out[j / 2] = pair(at.has(j) ? from.one(at.of(j)) : 0.0f, at.has(j + 1) ? from.one(at.of(j + 1)) : 0.0f);
    }
}
template <class T, bool kAligned, int G>
__device__ __forceinline__ void store_group(T* p, const Place<kAligned, G>& at, const Pair (&in)[G / 2]) {
    if constexpr (kAligned && sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(p + at.at) = make_uint4(narrow<T>(in[0]), narrow<T>(in[1]), narrow<T>(in[2]), narrow<T>(in[3]));
    } else {
        float v[G];
#pragma unroll
        for (int j = 0; j < G; j += 2) split(in[j / 2], &v[j], &v[j + 1]);
        if constexpr (kAligned) {
            *reinterpret_cast<float4*>(p + at.at) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < G; ++j)
                if (at.has(j)) p[at.of(j)] = from_f32<T>(v[j]);
        }
    }
}
// a gain: of the tensors' type, in 32 bits, or ones
template <class T, bool kAligned, int G>
__device__ __forceinline__ void load_gain(const void* p, bool f32, const Place<kAligned, G>& at, Pair (&out)[G / 2]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < G / 2; ++j) out[j] = pair(1.0f);
    } else if (!f32) {
        load_group<T, kAligned, G>(InMemory<T>{static_cast<const T*>(p)}, at, out);
    } else if constexpr (kAligned) {
#pragma unroll
        for (int j = 0; j < G; j += 4) {
            const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at.at + j);
            out[j / 2] = pair(x.x, x.y), out[j / 2 + 1] = pair(x.z, x.w);
        }
    } else {
        load_group<float, kAligned, G>(InMemory<float>{static_cast<const float*>(p)}, at, out);
    }
}

// Sums of K values (1 or up to 8) over the block's threads (whole warps, kWarps at most), for every thread.  Within a warp the values are
// dealt out while they are added, so that eight take nine exchanges and not forty.  `buf`: 8 floats a warp; two calls on it need a
// barrier between.
template <int kWarps, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float* buf) {
    constexpr int P = K == 1 ? 1 : 8;
    const unsigned lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    float w[P];
#pragma unroll
    for (int k = 0; k < P; ++k) w[k] = k < K ? v[k] : 0.0f;
#pragma unroll
    for (int o = 16, n = P / 2; o > 0; o >>= 1, n >>= 1) {
        if (n > 0) {
            const bool up = lane & o;
#pragma unroll
            for (int k = 0; k < n; ++k) {
                const float give = up ? w[k] : w[k + n];
                w[k] = (up ? w[k + n] : w[k]) + __shfl_xor_sync(0xffffffffu, give, o);
            }
        } else {
            w[0] += __shfl_xor_sync(0xffffffffu, w[0], o);
        }
    }
    // lane / (32 / P) says which value a lane has the warp's sum of
    if (lane % (32 / P) == 0) buf[(threadIdx.x >> 5) * P + lane / (32 / P)] = w[0];
    __syncthreads();
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; i += 32 / P)
        if (i + lane / P < warps) mine += buf[(i + lane / P) * P + lane % P];
#pragma unroll
    for (int o = P; o < 32; o <<= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = P == 1 ? mine : __shfl_sync(0xffffffffu, mine, k);
}

// How a kernel is laid out.  Slots: rows come through the ring and the values that all rows share (gains, a CHANNEL gate) stay in
// registers: with the ring in shared memory little first-level cache is left, and read for each row they would come from L2, as many
// bytes as the rows themselves.  Rows of more than 8192 values take 16 to a thread of 1024 and leave no registers for that, and
// some rows leave no room for two slots: they are read straight from global memory.
template <bool kAligned_, int kShare_, int kThreads_, int kBlocks_, bool kSlots_> struct Layout {
    static constexpr bool kAligned = kAligned_, kSlots = kSlots_;
    static constexpr int kShare = kShare_, kThreads = kThreads_, kBlocks = kBlocks_;
};
template <class T, class L> using From = std::conditional_t<L::kSlots, InSlot<T>, InMemory<T>>;
template <class T, class L, int N>
__device__ __forceinline__ From<T, L> row_from(const RowRing<T, N>& ring, const Source* src, int k, size_t row, unsigned slot) {
    if constexpr (L::kSlots) return {ring.template row_of<L::kAligned>(k, row, slot)};
    else return {reinterpret_cast<const T*>(src[k].p + row * src[k].ld)};
}

// Bound by HBM: x and y are read once, r and z written once.  Each block takes rows blockIdx.x, blockIdx.x + gridDim.x, ...
// Measured: 2048 x 4096 bf16, 18.3 us for 67 MB, of which about 10 are the copy's; the rest is the launch and the two sums that follow one
// another in each of a block's 7 rows.  16 values to a thread, two rows at once and three blocks to an SM came within 1 us.
template <class T, class L>
__global__ void __launch_bounds__(L::kThreads, L::kBlocks) block_norm_kernel(const __grid_constant__ NormArgs a) {
    constexpr int G = kGroup<T, L::kAligned>, NG = L::kShare / G;
    typedef Place<L::kAligned, G> At;
    extern __shared__ __align__(16) char memory[];
    __shared__ float sums[3 * 32];
    grid_release();
    const RowRing<T, 3> ring(a.src, a.cols, a.slots, a.slot_bytes, memory, a.flag);
    grid_wait();
    if (L::kSlots && threadIdx.x == 0)
        for (unsigned i = 0; i < a.slots && blockIdx.x + (size_t)i * gridDim.x < a.rows; ++i) ring.fetch(blockIdx.x + (size_t)i * gridDim.x, i);
    const bool branch = a.src[1].p != nullptr;
    const unsigned cols = (unsigned)a.cols;
    // the gain after the branch times a CHANNEL gate, and the gain before the next
    const auto load_e = [&](const At& at, Pair(&e)[G / 2]) {
        load_gain<T>(a.post_gain, a.gains_f32, at, e);
        if (a.gate_kind != ZKB_GATE_CHANNEL) return;
        Pair g[G / 2];
        load_gain<T>(a.gate, a.gains_f32, at, g);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) e[j] = e[j] * g[j];
    };
    Pair held_e[L::kSlots ? NG : 1][G / 2], held_w[L::kSlots ? NG : 1][G / 2];
    if constexpr (L::kSlots) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const At at(g, cols);
            if (!at.any()) continue;
            load_e(at, held_e[g]);
            load_gain<T>(a.pre_gain, a.gains_f32, at, held_w[g]);
        }
    }
    unsigned slot = 0, odd = 0;
    uint32_t phase = 0;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (L::kSlots) ring.wait(slot, phase);
        Pair x[NG][G / 2], y[NG][G / 2], s2 = pair(0.0f);
        float s[1];
        const auto from_x = row_from<T, L>(ring, a.src, 0, row, slot), from_y = row_from<T, L>(ring, a.src, 1, row, slot),
                   from_gate = row_from<T, L>(ring, a.src, 2, row, slot);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const At at(g, cols);
#pragma unroll
            for (int j = 0; j < G / 2; ++j) x[g][j] = y[g][j] = pair(0.0f);
            if (!at.any()) continue;
            load_group<T>(from_x, at, x[g]);
            if (!branch) continue;
            load_group<T>(from_y, at, y[g]);
#pragma unroll
            for (int j = 0; j < G / 2; ++j) s2 = fma(y[g][j], y[g][j], s2);
        }
        float post_inv = 1.0f;
        if (a.post_norm) {
            s[0] = total(s2);
            row_sums<L::kThreads / 32, 1>(s, sums);
            post_inv = rsqrtf(s[0] * a.one_over_cols + a.eps);
            if (threadIdx.x == 0 && a.post_inv) a.post_inv[row] = post_inv;
        }
        s2 = pair(0.0f);
        T* const r_row = static_cast<T*>(a.r) + row * a.ldr;
        const Pair by = pair(a.scale * post_inv * (a.gate_kind == ZKB_GATE_ROW ? to_f32<T>(static_cast<const T*>(a.gate)[row]) : 1.0f));
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const At at(g, cols);
            if (!at.any()) continue;
            if (branch) {
                Pair w[G / 2];
                if constexpr (!L::kSlots) load_e(at, w);
#pragma unroll
                for (int j = 0; j < G / 2; ++j) y[g][j] = y[g][j] * (L::kSlots ? held_e[L::kSlots ? g : 0][j] : w[j]);
                if (a.gate_kind == ZKB_GATE_ELEMENT) {
                    load_group<T>(from_gate, at, w);
#pragma unroll
                    for (int j = 0; j < G / 2; ++j) y[g][j] = y[g][j] * w[j];
                }
#pragma unroll
                for (int j = 0; j < G / 2; ++j) x[g][j] = fma(y[g][j], by, x[g][j]);
            }
            if (a.r) store_group<T>(r_row, at, x[g]);
#pragma unroll
            for (int j = 0; j < G / 2; ++j) s2 = fma(x[g][j], x[g][j], s2);
        }
        s[0] = total(s2);
        row_sums<L::kThreads / 32, 1>(s, sums + 32 + 32 * odd);      // behind its barrier every thread has read this row's slot
        odd ^= 1;
        if (L::kSlots) {
            const size_t next = row + (size_t)a.slots * gridDim.x;
            if (threadIdx.x == 0 && next < a.rows) ring.fetch(next, slot);
            if (++slot == a.slots) { slot = 0; phase ^= 1; }
        }
        if (!a.pre_norm) continue;
        const float inv = rsqrtf(s[0] * a.one_over_cols + a.eps);
        if (threadIdx.x == 0 && a.pre_inv) a.pre_inv[row] = inv;
        if (!a.z) continue;
        T* const z_row = static_cast<T*>(a.z) + row * a.ldz;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const At at(g, cols);
            if (!at.any()) continue;
            Pair w[G / 2];
            if constexpr (!L::kSlots) load_gain<T>(a.pre_gain, a.gains_f32, at, w);
#pragma unroll
            for (int j = 0; j < G / 2; ++j) w[j] = (L::kSlots ? held_w[L::kSlots ? g : 0][j] : w[j]) * (x[g][j] * pair(inv));
            store_group<T>(z_row, at, w);
        }
    }
    ring.close();
}

// The gradients.  With p = dz w_pre, the gradient of r is d = dr + inv (p - r b), b = inv^2 mean(p r); with e = gate w_post, that of y
// is a ip (e d - y ip^2 mean(e d y)).  The last mean needs no pass of its own: by the first formula sum(e d y) =
// sum(e y dr) + inv sum(e y p) - inv b sum(e y r), so that one round of six sums serves both norms.
//
// Two sums over rows serve all three vectors: dz r inv gives the gain before the next branch, and S = d y ip (times the gate where
// that differs from row to row) both the other gain, a gate S, and a CHANNEL gate, a w_post S.  Each block keeps its rows'
// share of them in registers; norm_reduce_kernel adds the shares in the order of the blocks, so that a result does not depend on timing.
//
// Measured: 8192 x 5120 bf16 with f32 gains, 116 us (120 with the reduction) for 503 MB, 64% of the copy rate.  Bound by the shared-memory
// and shuffle pipe and the row's dependent chain rather than by HBM: without the sums it takes 101 us, with the loads alone 81.
// Before: gains read for each row (from L2, there is little first-level cache beside the ring) 168 us; two rows at once 135 us; the
// sums of the next row formed beside this one's end 137 us; 16 values to a thread of 320 141 us.
template <class T, class L>
__global__ void __launch_bounds__(L::kThreads, L::kBlocks) block_norm_backward_kernel(const __grid_constant__ NormGradArgs a) {
    constexpr int G = kGroup<T, L::kAligned>, NG = L::kShare / G;
    typedef Place<L::kAligned, G> At;
    extern __shared__ __align__(16) char memory[];
    __shared__ float sums[2][8 * 32];
    grid_release();
    const RowRing<T, 5> ring(a.src, a.cols, a.slots, a.slot_bytes, memory, a.flag);
    grid_wait();
    if (L::kSlots && threadIdx.x == 0)
        for (unsigned i = 0; i < a.slots && blockIdx.x + (size_t)i * gridDim.x < a.rows; ++i) ring.fetch(blockIdx.x + (size_t)i * gridDim.x, i);
    const bool branch = a.src[2].p != nullptr, more = a.src[3].p != nullptr, element = a.gate_kind == ZKB_GATE_ELEMENT;
    const unsigned cols = (unsigned)a.cols;
    // the gain after the branch times a CHANNEL gate
    const auto load_e = [&](const At& at, Pair(&e)[G / 2]) {
        load_gain<T>(a.post_gain, a.gains_f32, at, e);
        if (a.gate_kind != ZKB_GATE_CHANNEL) return;
        Pair g[G / 2];
        load_gain<T>(a.gate, a.gains_f32, at, g);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) e[j] = e[j] * g[j];
    };
    Pair acc_pre[NG][G / 2], acc_post[NG][G / 2], held_e[L::kSlots ? NG : 1][G / 2], held_w[L::kSlots ? NG : 1][G / 2];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int j = 0; j < G / 2; ++j) acc_pre[g][j] = acc_post[g][j] = pair(0.0f);
        const At at(g, cols);
        if (!L::kSlots || !at.any()) continue;
        load_e(at, held_e[L::kSlots ? g : 0]);
        load_gain<T>(a.pre_gain, a.gains_f32, at, held_w[L::kSlots ? g : 0]);
    }
    const auto pre_gain = [&](int g, const At& at, Pair(&w)[G / 2]) {
        if constexpr (!L::kSlots) load_gain<T>(a.pre_gain, a.gains_f32, at, w);
        else
#pragma unroll
            for (int j = 0; j < G / 2; ++j) w[j] = held_w[g][j];
    };
    const auto post_gain = [&](int g, const At& at, Pair(&w)[G / 2]) {
        if constexpr (!L::kSlots) load_e(at, w);
        else
#pragma unroll
            for (int j = 0; j < G / 2; ++j) w[j] = held_e[g][j];
    };
    unsigned slot = 0, odd = 0, done = 0;   // done: the slot of the row before
    uint32_t phase = 0;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (L::kSlots) ring.wait(slot, phase);
        const auto from_r = row_from<T, L>(ring, a.src, 0, row, slot), from_dz = row_from<T, L>(ring, a.src, 1, row, slot),
                   from_y = row_from<T, L>(ring, a.src, 2, row, slot), from_dr = row_from<T, L>(ring, a.src, 3, row, slot),
                   from_gate = row_from<T, L>(ring, a.src, 4, row, slot);
        Pair rr = pair(0.0f), pr = rr, yy = rr, eyd = rr, eyp = rr, eyr = rr;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const At at(g, cols);
            if (!at.any()) continue;
            Pair r[G / 2], p[G / 2], w[G / 2];
            if (a.pre_norm) {
                load_group<T>(from_r, at, r);
                load_group<T>(from_dz, at, p);
                pre_gain(g, at, w);
#pragma unroll
                for (int j = 0; j < G / 2; ++j) {
                    p[j] = p[j] * w[j];
                    rr = fma(r[j], r[j], rr);
                    pr = fma(p[j], r[j], pr);
                }
            }
            if (branch) {
                Pair y[G / 2];
                load_group<T>(from_y, at, y);
                post_gain(g, at, w);
#pragma unroll
                for (int j = 0; j < G / 2; ++j) {
                    yy = fma(y[j], y[j], yy);
                    y[j] = y[j] * w[j];
                }
                if (element) {
                    load_group<T>(from_gate, at, w);
#pragma unroll
                    for (int j = 0; j < G / 2; ++j) y[j] = y[j] * w[j];
                }
                if (a.pre_norm)
#pragma unroll
                    for (int j = 0; j < G / 2; ++j) {
                        eyp = fma(y[j], p[j], eyp);
                        eyr = fma(y[j], r[j], eyr);
                    }
                if (more) {
                    load_group<T>(from_dr, at, w);
#pragma unroll
                    for (int j = 0; j < G / 2; ++j) eyd = fma(y[j], w[j], eyd);
                }
            }
        }
        float s[6] = {total(rr), total(pr), total(yy), total(eyd), total(eyp), total(eyr)};
        row_sums<L::kThreads / 32, 6>(s, sums[odd]);
        odd ^= 1;
        if (L::kSlots) {   // behind the barrier in row_sums every thread is done with the row before
            if (threadIdx.x == 0 && row >= gridDim.x) {
                const size_t next = row + (size_t)(a.slots - 1) * gridDim.x;
                if (next < a.rows) ring.fetch(next, done);
            }
            done = slot;
            if (++slot == a.slots) { slot = 0; phase ^= 1; }
        }
        const float inv = a.pre_norm ? rsqrtf(s[0] * a.one_over_cols + a.eps) : 0.0f, b = inv * inv * s[1] * a.one_over_cols;
        const float post_inv = a.post_norm ? rsqrtf(s[2] * a.one_over_cols + a.eps) : 1.0f;
        const float edy = s[3] + inv * (s[4] - b * s[5]);
        // a ROW gate is not in e: it scales the whole branch
        const float row_gate = a.gate_kind == ZKB_GATE_ROW ? to_f32<T>(static_cast<const T*>(a.gate)[row]) : 1.0f;
        if (a.want_gate && a.gate_kind == ZKB_GATE_ROW && threadIdx.x == 0) static_cast<T*>(a.dgate)[row] = from_f32<T>(a.scale * post_inv * edy);
        const float by = a.scale * row_gate * post_inv;
        const Pair by2 = pair(by), less = pair(a.post_norm ? -by * post_inv * post_inv * edy * a.one_over_cols : 0.0f), inv2 = pair(inv), b2 = pair(-b);
        const Pair share = pair(post_inv * row_gate), dg_by = pair(a.scale * post_inv);
        T* const dx_row = static_cast<T*>(a.dx) + row * a.lddx;
        T* const dy_row = static_cast<T*>(a.dy) + row * a.lddy;
        T* const dgate_row = static_cast<T*>(a.dgate) + row * a.lddgate;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const At at(g, cols);
            if (!at.any()) continue;
            Pair d[G / 2], w[G / 2];
#pragma unroll
            for (int j = 0; j < G / 2; ++j) d[j] = pair(0.0f);
            if (more) load_group<T>(from_dr, at, d);
            if (a.pre_norm) {
                Pair r[G / 2], dz[G / 2];
                load_group<T>(from_r, at, r);
                load_group<T>(from_dz, at, dz);
                pre_gain(g, at, w);
#pragma unroll
                for (int j = 0; j < G / 2; ++j) {
                    acc_pre[g][j] = fma(dz[j] * r[j], inv2, acc_pre[g][j]);
                    d[j] = fma(fma(r[j], b2, dz[j] * w[j]), inv2, d[j]);
                }
            }
            if (a.dx) store_group<T>(dx_row, at, d);
            if (!branch) continue;
            Pair y[G / 2];
            load_group<T>(from_y, at, y);
            post_gain(g, at, w);
            if (element) {
                Pair gate[G / 2], dy[G / 2];
                load_group<T>(from_gate, at, gate);
#pragma unroll
                for (int j = 0; j < G / 2; ++j) {
                    dy[j] = d[j] * y[j];
                    acc_post[g][j] = fma(dy[j] * gate[j], share, acc_post[g][j]);
                    dy[j] = dy[j] * (w[j] * dg_by);
                    w[j] = w[j] * gate[j];
                }
                if (a.want_gate) store_group<T>(dgate_row, at, dy);
            } else {
#pragma unroll
                for (int j = 0; j < G / 2; ++j) acc_post[g][j] = fma(d[j] * y[j], share, acc_post[g][j]);
            }
            if (a.dy) {
#pragma unroll
                for (int j = 0; j < G / 2; ++j) d[j] = fma(d[j] * w[j], by2, y[j] * less);
                store_group<T>(dy_row, at, d);
            }
        }
    }
    ring.close();
    if (!a.partial) return;
    float* out = a.partial + (size_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const At at(g, cols);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) {
            float v[2], u[2];
            split(acc_pre[g][j], &v[0], &v[1]);
            split(acc_post[g][j], &u[0], &u[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (at.any() && at.has(2 * j + k)) {
                    out[at.of(2 * j + k)] = v[k];
                    out[a.cols + at.of(2 * j + k)] = u[k];
                }
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
        const auto one = [&](const void* p) { return !p ? 1.0f : a.gains_f32 ? static_cast<const float*>(p)[c] : to_f32<T>(static_cast<const T*>(p)[c]); };
        put(a.dpost, a.scale * one(a.gate) * s);
        put(a.dgate, a.scale * one(a.post_gain) * s);
    }
}

// threads to a row for `per` values a thread, whole warps
unsigned row_threads(size_t cols, unsigned per) { return std::max(32u, div_up(div_up(cols, per), 32) * 32); }

constexpr size_t kRingHead = 16 * 8;
// Places the matrices in a slot; returns its bytes.
template <class Args> size_t lay_slot(Args* a, int matrices, size_t es) {
    size_t slot = 0;
    for (int k = 0; k < matrices; ++k) {
        a->src[k].at = (unsigned)slot;
        if (a->src[k].p) slot += slot_row_bytes(a->cols, es);
    }
    a->slot_bytes = (unsigned)slot;
    return std::max<size_t>(slot, 16);
}
// The most that a block may ask for beside its sums when there are that many on an SM; of its share, 1 KB is the system's and up to 3 KB the sums'.
constexpr size_t ring_share(int blocks_per_sm) { return 224 * 1024 / blocks_per_sm - 4096; }
size_t slots_for(size_t slot, int blocks_per_sm) { return std::min<size_t>(8, (ring_share(blocks_per_sm) - kRingHead) / slot); }

// The grid of a kernel over rows, and its ring: as many blocks as are resident, each with as many slots as fit.
template <class L, class Kernel, class Args>
int plan_rows(Kernel kernel, unsigned threads, Args* a, unsigned* blocks, size_t* smem) {
    int resident = 0;
    ZKB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, threads, kRingHead));
    resident = std::max(1, resident);
    *smem = kRingHead;
    if (L::kSlots) {
        const size_t slot = std::max(a->slot_bytes, 16u);
        while (resident > 1 && slots_for(slot, resident) < 3) --resident;
        a->slots = (unsigned)slots_for(slot, resident);
        *smem += a->slots * slot;
        // The limit belongs to the kernel, which calls of other widths run too, perhaps from another thread between this line and the
        // launch: it is always the most that any of them asks for, never this call's size.
        ZKB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring_share(1)));
    }
    *blocks = (unsigned)std::min<size_t>(a->rows, (size_t)resident * sm_count());
    return ZKB_OK;
}

template <class T, class L>
int norm_launch(NormArgs a, cudaStream_t s) {
    const unsigned threads = row_threads(a.cols, L::kShare);
    const auto kernel = block_norm_kernel<T, L>;
    unsigned blocks;
    size_t smem;
    ZKB_TRY((plan_rows<L>(kernel, threads, &a, &blocks, &smem)));
    return launch_beside("block_norm", kernel, blocks, threads, smem, s, a);
}
template <class T, bool kAligned>
int norm_launch(NormArgs a, cudaStream_t s) {
    // 32 M values of bf16 (f32), a CHANNEL gate: 4096 columns 53.5 us (97) in the first, 52.5 (97) in the second; 8192 columns 56 (98) in the
    // second, 77 (117) in the third, which takes 96 (151) for 13824
    lay_slot(&a, 3, sizeof(T));
    if (a.cols <= 4096) return norm_launch<T, Layout<kAligned, 8, 512, 2, true>>(a, s);
    if (a.cols <= 8192) return norm_launch<T, Layout<kAligned, 8, 1024, 1, true>>(a, s);
    return norm_launch<T, Layout<kAligned, 16, 1024, 1, false>>(a, s);
}

template <class T, class L>
int norm_backward_launch(NormGradArgs a, void* dpost, void* dpre, cudaStream_t s) {
    const unsigned threads = row_threads(a.cols, L::kShare);
    const auto kernel = block_norm_backward_kernel<T, L>;
    unsigned blocks;
    size_t smem;
    ZKB_TRY((plan_rows<L>(kernel, threads, &a, &blocks, &smem)));
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
template <class T, bool kAligned>
int norm_backward_launch(NormGradArgs a, void* dpost, void* dpre, cudaStream_t s) {
    // The same 32 M values: 2560 columns 99.5 us (166) in the first, 101 (167) in the second; 5120 columns 101 (180) in the second, 119 (176)
    // in the third; 8192 bf16 columns 96 in the third, 197 in the fourth, which spills and reads rows twice: 303 for 8192 f32 columns, 233
    // (339) for 13824.
    const bool slots = slots_for(lay_slot(&a, 5, sizeof(T)), 1) >= 2;   // the present row and one on its way
    if (slots && a.cols <= 2560) return norm_backward_launch<T, Layout<kAligned, 8, 320, 2, true>>(a, dpost, dpre, s);
    if (slots && a.cols <= 5120) return norm_backward_launch<T, Layout<kAligned, 8, 640, 1, true>>(a, dpost, dpre, s);
    if (slots && a.cols <= 8192) return norm_backward_launch<T, Layout<kAligned, 16, 512, 1, true>>(a, dpost, dpre, s);
    return norm_backward_launch<T, Layout<kAligned, 16, 1024, 1, false>>(a, dpost, dpre, s);
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
    if (m.ld < cols && rows > 1) return fail(ZKB_ERR_DIM, std::string(who) + ": " + m.name + ": row stride below the row's length");
    ZKB_TRY(check_device(m.p, type_size(dtype), who, m.name));
    if (!aligned_to(m.p, 16) || (m.ld * type_size(dtype)) % 16) *wide = false;
    return ZKB_OK;
}
int check_vector(const char* who, const void* p, const char* name, int dtype, bool* wide) {
    if (!p) return ZKB_OK;
    ZKB_TRY(check_device(p, type_size(dtype), who, name));
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
    a.scale = residual_scale, a.eps = eps, a.one_over_cols = (float)(1.0 / (double)cols), a.gate_kind = gate_kind;
    a.post_norm = post_norm != 0, a.pre_norm = pre_norm != 0, a.gains_f32 = gains_dtype == ZKB_F32;
    if (!(a.flag = tc::wait_flag())) return ZKB_ERR_CUDA;
    const cudaStream_t s = as_stream(stream);
    if (dtype == ZKB_F32) return wide ? norm_launch<float, true>(a, s) : norm_launch<float, false>(a, s);
    if (dtype == ZKB_F16) return wide ? norm_launch<__half, true>(a, s) : norm_launch<__half, false>(a, s);
    return wide ? norm_launch<bf16, true>(a, s) : norm_launch<bf16, false>(a, s);
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
    a.scale = residual_scale, a.eps = eps, a.one_over_cols = (float)(1.0 / (double)cols), a.gate_kind = gate_kind;
    a.post_norm = post_norm != 0, a.pre_norm = pre_norm != 0, a.gains_f32 = gains_dtype == ZKB_F32, a.want_gate = d_dgate != nullptr;
    if (!(a.flag = tc::wait_flag())) return ZKB_ERR_CUDA;
    if (dtype == ZKB_F32) return wide ? norm_backward_launch<float, true>(a, d_dpost_gain, d_dpre_gain, s) : norm_backward_launch<float, false>(a, d_dpost_gain, d_dpre_gain, s);
    if (dtype == ZKB_F16) return wide ? norm_backward_launch<__half, true>(a, d_dpost_gain, d_dpre_gain, s) : norm_backward_launch<__half, false>(a, d_dpost_gain, d_dpre_gain, s);
    return wide ? norm_backward_launch<bf16, true>(a, d_dpost_gain, d_dpre_gain, s) : norm_backward_launch<bf16, false>(a, d_dpost_gain, d_dpre_gain, s);
}

}  // extern "C"
