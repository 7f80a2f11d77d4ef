// The gated feed-forward block up to its product: h = act(x Wg) * (x Wu), and the gradients of x, Wg and Wu.
//
// Weights are [in, hidden], as zkFC and FrTensor::matmul take them.  Sums are in 32 bits; h is formed from the unrounded sums.
#include <algorithm>
#include <initializer_list>
#include <utility>

#include "tensorcore.cuh"

namespace zkb {
namespace {

// act(g) and, for the gradient, its derivative.  1 / (1 + exp) by the approximate quotient (2^-22), which is far below a 16-bit step.
template <int kAct, bool kDerivative>
__device__ __forceinline__ float activate(float g, float* d) {
    if constexpr (kAct == ZKB_ACT_SILU) {
        const float s = __fdividef(1.0f, 1.0f + __expf(-g));
        if (kDerivative) *d = s * (1.0f + g * (1.0f - s));
        return g * s;
    } else if constexpr (kAct == ZKB_ACT_GELU) {
        const float c = 0.5f * erfcf(g * -0.70710678118654752f);   // 1 + erf would cancel below zero
        if (kDerivative) *d = c + g * __expf(-0.5f * g * g) * 0.39894228040143268f;
        return g * c;
    } else if constexpr (kAct == ZKB_ACT_GELU_TANH) {
        // (1 + tanh k) / 2 = 1 / (1 + exp(-2k))
        const float k = 0.79788456080286536f * (g + 0.044715f * g * g * g);
        const float s = __fdividef(1.0f, 1.0f + __expf(-2.0f * k));
        // far out s (1 - s) is zero, and stays so beside a square that would pass 32 bits
        if (kDerivative) *d = s + 2.0f * g * s * (1.0f - s) * 0.79788456080286536f * (1.0f + 0.134145f * fminf(g * g, 1e30f));
        return g * s;
    } else {
        if (kDerivative) *d = g > 0.0f ? 1.0f : 0.0f;
        return g > 0.0f ? g : g != g ? g : 0.0f;
    }
}
// h = act(g) * u in place of g
template <int kAct, int N>
__device__ __forceinline__ void gate_by(float (&g)[N], const float (&u)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = activate<kAct, false>(g[i], nullptr) * u[i];
}
template <int N>
__device__ __forceinline__ void gate(int act, float (&g)[N], const float (&u)[N]) {
    if (act == ZKB_ACT_SILU) gate_by<ZKB_ACT_SILU>(g, u);
    else if (act == ZKB_ACT_GELU) gate_by<ZKB_ACT_GELU>(g, u);
    else if (act == ZKB_ACT_GELU_TANH) gate_by<ZKB_ACT_GELU_TANH>(g, u);
    else gate_by<ZKB_ACT_RELU>(g, u);
}
// the gradients of g and u, in their places, from that of h
template <int kAct, int N>
__device__ __forceinline__ void ungate_by(float (&g)[N], float (&u)[N], const float (&dh)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float da;
        const float a = activate<kAct, true>(g[i], &da);
        g[i] = dh[i] * u[i] * da;
        u[i] = dh[i] * a;
    }
}
template <int N>
__device__ __forceinline__ void ungate(int act, float (&g)[N], float (&u)[N], const float (&dh)[N]) {
    if (act == ZKB_ACT_SILU) ungate_by<ZKB_ACT_SILU>(g, u, dh);
    else if (act == ZKB_ACT_GELU) ungate_by<ZKB_ACT_GELU>(g, u, dh);
    else if (act == ZKB_ACT_GELU_TANH) ungate_by<ZKB_ACT_GELU_TANH>(g, u, dh);
    else ungate_by<ZKB_ACT_RELU>(g, u, dh);
}

// ---- the product kernel -----------------------------------------------------------------------------------------------------
//
// Bound by the tensor cores.  Persistent pairs of blocks (one block per SM) work through 256 x 256 tiles.  Each block holds 128 rows of the
// first operand and 128 columns of the second, so that a slice costs both SMs together 64 KB of copies and shared memory where two
// blocks on their own would need 96.  In each block warp 0 copies 64-deep slices into a ring; in the first, warp 1 issues
// the products (256 x 256 x 16 each) into one of two accumulators in tensor memory; warps 4 to 11 of both take their 128 rows of the other
// accumulator out, so that a tile's epilogue runs beside the next tile's products.
//
// Measured: 2048 x 4096 x 11008 bf16, 300 to 310 us call after call under the power limit (1.2 PFLOP/s; torch's two products alone 259 to
// 265 us), 238 for a single launch after idling, the tensor pipe busy 87% of the time; gradients 560 to 620 us, 520 at best.  One block to a tile of 128 x 256 took 360 us; a switch over the
// activation inside the epilogue's loop 337; the gradients' two kinds of tiles in a launch each 10% more.  Fetching slices ahead into L2 only cost.
//
// The forms of a tile:
//   gated    first operand x; second the two weights side by side, 128 columns of each in a tile; result act(g) * u
//   summed   dg, then du; w_gate, then w_up: one sum over both; result dx
//   paired   x^T; dg for the first half of the tiles, du for the second; results dw_gate and dw_up
// The gradients' launch holds tiles of both of the last: the few, long tiles of dx first, one or two to a pair of blocks, and the
// many short ones of the weights where there is room.  The pairs with one tile of dx less take `head` of the short ones each before
// the rest are dealt out to all, so that all end together.  Where dx has fewer tiles than there are pairs, each of its sums is cut
// into parts, which are left in 32 bits and added in order by glu_after_kernel.
constexpr int kTile = 256, kHalf = 128, kDepth = 64;
constexpr int kTakers = 8;             // epilogue warps of a block, two to 32 rows: with 4 a tile of few slices waits for its way out
constexpr int kProductThreads = 128 + 32 * kTakers;
constexpr int kStageBytes = 32 * 80;   // an epilogue warp's 32 x 32 values on their way out, rows 80 bytes apart
constexpr int kRing = 6, kSlice = 2 * kHalf * kDepth * 2;
constexpr size_t kProductSmem = 1024 + (size_t)kRing * kSlice + kTakers * kStageBytes + 256;

struct Results {
    unsigned m, n;                           // of one result (gated: hidden)
    unsigned row_tiles, col_tiles, slices;   // its tiles, and slices of 64 of one sum
    void* out[3];                            // gated: h, gate, up (or null); summed: dx; paired: dw_gate, dw_up
    size_t ld[3];                            // addresses and row strides are whole 16 bytes
};
struct GatedArgs {
    CUtensorMap a, b[2];
    Results r;
    int act;
    int* flag;
};
struct GradArgs {
    CUtensorMap dg_rows[2], w[2];            // summed: dg and du in boxes of 128 rows, the weights
    CUtensorMap x, dg_cols[2];               // paired: x, dg and du in boxes of 64 rows
    Results dx, dw;
    unsigned head, parts;                    // parts: of dx's sums
    float* sums;                             // [parts][m][sums_ld], if there are several
    unsigned sums_ld;
    const float* unscale;                    // f16: what the sums are multiplied by
    int* flag;
};
struct Tile { unsigned row, col, pair, part, from, to; bool paired; };   // from, to: its slices

// 32 x 32 values of a warp (row i with lane i) to rows row0.. and columns col0.. of a matrix of m x n.
template <class T>
__device__ __forceinline__ void store_block(char* stage, const float (&v)[32], T* out, size_t ld, unsigned row0, unsigned col0, unsigned m, unsigned n) {
    const unsigned lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        Vec<T, 8> x;
#pragma unroll
        for (int j = 0; j < 8; ++j) x.v[j] = from_f32<T>(v[i + j]);
        *reinterpret_cast<Vec<T, 8>*>(stage + lane * 80 + i * 2) = x;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned r = i * 8 + lane / 4, c = (lane % 4) * 8;
        const Vec<T, 8> x = *reinterpret_cast<const Vec<T, 8>*>(stage + r * 80 + c * 2);
        if (row0 + r >= m) continue;
        T* to = out + (size_t)(row0 + r) * ld + col0 + c;
        if (col0 + c + 8 <= n) {
            *reinterpret_cast<Vec<T, 8>*>(to) = x;
        } else {
            for (unsigned j = 0; col0 + c + j < n && j < 8; ++j) to[j] = x.v[j];
        }
    }
    __syncwarp();
}

// Tile number to its row and column: rows first within bands of 16 rows of tiles, so that the blocks at work at one time share
// both operands in L2.
__device__ __forceinline__ void tile_place(unsigned tile, unsigned row_tiles, unsigned col_tiles, unsigned* row, unsigned* col) {
    const unsigned band = tile / (16 * col_tiles), in = tile % (16 * col_tiles);
    const unsigned height = min(16u, row_tiles - band * 16);
    *row = band * 16 + in % height;
    *col = in / height;
}

// The i-th tile of a pair of blocks; false behind its last.
__device__ __forceinline__ const Results& results_of(const GatedArgs& p, const Tile&) { return p.r; }
__device__ __forceinline__ const Results& results_of(const GradArgs& p, const Tile& t) { return t.paired ? p.dw : p.dx; }
__device__ __forceinline__ bool tile_of(const GatedArgs& p, unsigned i, unsigned me, unsigned pairs, Tile* t) {
    const unsigned n = me + i * pairs;
    if (n >= p.r.row_tiles * p.r.col_tiles) return false;
    t->pair = t->part = t->from = 0, t->to = p.r.slices, t->paired = false;
    tile_place(n, p.r.row_tiles, p.r.col_tiles, &t->row, &t->col);
    return true;
}
__device__ __forceinline__ bool tile_of(const GradArgs& p, unsigned i, unsigned me, unsigned pairs, Tile* t) {
    const unsigned whole = p.dx.row_tiles * p.dx.col_tiles, longs = whole * p.parts, more = longs % pairs, mine = longs / pairs + (me < more);
    const unsigned per = p.dw.row_tiles * p.dw.col_tiles;
    t->pair = t->part = 0, t->paired = i >= mine;
    if (!t->paired) {
        const unsigned n = me + i * pairs;
        t->part = n / whole;
        t->from = 2 * p.dx.slices * t->part / p.parts, t->to = 2 * p.dx.slices * (t->part + 1) / p.parts;
        tile_place(n % whole, p.dx.row_tiles, p.dx.col_tiles, &t->row, &t->col);
        return true;
    }
    i -= mine;
    unsigned n;
    const unsigned ahead = more ? p.head : 0;
    if (me >= more && i < ahead) n = me - more + i * (pairs - more);
    else n = ahead * (pairs - more) + me + (i - (me >= more ? ahead : 0)) * pairs;
    if (n >= 2 * per) return false;
    t->pair = n / per;
    t->from = 0, t->to = p.dw.slices;
    tile_place(n % per, p.dw.row_tiles, p.dw.col_tiles, &t->row, &t->col);
    return true;
}

template <class T, class Args>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kProductThreads) glu_product_kernel(const __grid_constant__ Args p) {
    constexpr bool kGated = std::is_same<Args, GatedArgs>::value;
    constexpr int kA = kHalf * kDepth * 2;
    extern __shared__ char raw[];
    char* ring = raw + ((1024 - (tc::smem_address(raw) & 1023)) & 1023);
    char* stages = ring + kRing * kSlice;
    uint64_t* bars = reinterpret_cast<uint64_t*>(stages + kTakers * kStageBytes);
    volatile int* dead = reinterpret_cast<volatile int*>(bars + 2 * kRing + 4);
    const uint32_t full = tc::smem_address(bars), empty = full + 8 * kRing, ready = empty + 8 * kRing, taken = ready + 16;
    const uint32_t tmem_at = taken + 24;
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = tc::cluster_rank();
    const tc::Watch watch = {dead, p.flag};
    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) {
            tc::barrier_init(full + 8 * i, 1);
            tc::barrier_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::barrier_init(ready + 8 * i, 1);
            tc::barrier_init(taken + 8 * i, 2 * kTakers);   // the epilogue warps of both blocks
        }
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 2) tc::tmem_alloc_pair(tmem_at, 2 * kTile);
    tc::fence_before_sync();
    __syncthreads();
    tc::cluster_barrier();
    tc::fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(bars + 2 * kRing + 5);

    const unsigned first = blockIdx.x / 2, step = gridDim.x / 2;
    if (warp == 0 && lane == 0) {
        unsigned at = 0;
        uint32_t phase = 0;
        bool fine = true;
        Tile t;
        for (unsigned i = 0; fine && tile_of(p, i, first, step, &t); ++i) {
            const unsigned m = t.row * kTile + rank * kHalf, n = t.col * kTile + rank * kHalf;
            const Results& r = results_of(p, t);
            for (unsigned s = t.from; s < t.to; ++s) {
                if (!tc::barrier_wait(empty + 8 * at, phase ^ 1, watch)) { fine = false; break; }
                const uint32_t a = tc::smem_address(ring) + at * kSlice, b = a + kA, bar = tc::address_in(full + 8 * at, 0);
                if (rank == 0) tc::barrier_expect(full + 8 * at, 2 * kSlice);
                const unsigned sum = s >= r.slices;
                const int k = (s - sum * r.slices) * kDepth;
                if constexpr (kGated) {   // the first block holds w_gate's columns, the second w_up's
                    tc::load_box_pair(&p.a, a, bar, k, m);
                    tc::load_box_pair(&p.b[rank], b, bar, t.col * kHalf, k);
                    tc::load_box_pair(&p.b[rank], b + 8192, bar, t.col * kHalf + 64, k);
                } else if (t.paired) {
                    tc::load_box_pair(&p.x, a, bar, m, k);
                    tc::load_box_pair(&p.x, a + 8192, bar, m + 64, k);
                    tc::load_box_pair(&p.dg_cols[t.pair], b, bar, n, k);
                    tc::load_box_pair(&p.dg_cols[t.pair], b + 8192, bar, n + 64, k);
                } else {
                    tc::load_box_pair(&p.dg_rows[sum], a, bar, k, m);
                    tc::load_box_pair(&p.w[sum], b, bar, k, n);
                }
                if (++at == kRing) { at = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        unsigned at = 0;
        uint32_t phase = 0;
        bool fine = true;
        Tile t;
        for (unsigned i = 0; fine && tile_of(p, i, first, step, &t); ++i) {
            const unsigned acc = i & 1;
            if (!tc::barrier_wait(taken + 8 * acc, ((i >> 1) & 1) ^ 1, watch)) break;
            tc::fence_after_sync();
            const bool a_mn = !kGated && t.paired, b_mn = kGated || t.paired;
            const uint32_t instruction = tc::instruction<T>(kTile, kTile, a_mn, b_mn), a_step = a_mn ? 2048 : 32, b_step = b_mn ? 2048 : 32;
            for (unsigned s = t.from; s < t.to; ++s) {
                if (!tc::barrier_wait(full + 8 * at, phase, watch)) { fine = false; break; }
                tc::fence_after_sync();
                const uint32_t a = tc::smem_address(ring) + at * kSlice, b = a + kA;
#pragma unroll
                for (int k = 0; k < kDepth / 16; ++k)
                    tc::product_pair(tmem + acc * kTile, tc::tile_descriptor(a + k * a_step, a_mn, 8192), tc::tile_descriptor(b + k * b_step, b_mn, 8192),
                                     instruction, s > t.from || k);
                tc::commit_pair(empty + 8 * at);
                if (++at == kRing) { at = 0; phase ^= 1; }
            }
            if (fine) tc::commit_pair(ready + 8 * acc);
        }
    } else if (warp >= 4) {
        char* stage = stages + (warp - 4) * kStageBytes;
        const unsigned side = (warp - 4) / 4;
        constexpr bool kScaled = !kGated && std::is_same<T, __half>::value;
        float unscale = 1.0f;
        if constexpr (kScaled) unscale = *p.unscale;
        Tile t;
        for (unsigned i = 0; tile_of(p, i, first, step, &t); ++i) {
            const unsigned acc = i & 1;
            if (!tc::barrier_wait_warp(ready + 8 * acc, (i >> 1) & 1, watch)) break;
            tc::fence_after_sync();
            const uint32_t from = tmem + (warp % 4 * 32 << 16) + acc * kTile;
            const unsigned row0 = t.row * kTile + rank * kHalf + warp % 4 * 32;
            const Results& r = results_of(p, t);
            if constexpr (kGated) {
                for (unsigned c = side * (kHalf / 2); c < (side + 1) * (kHalf / 2); c += 32) {
                    float g[32], u[32];
                    tc::load_columns(from + c, g);
                    tc::load_columns(from + kHalf + c, u);
                    const unsigned col0 = t.col * kHalf + c;
                    if (r.out[1]) {
                        store_block<T>(stage, g, static_cast<T*>(r.out[1]), r.ld[1], row0, col0, r.m, r.n);
                        store_block<T>(stage, u, static_cast<T*>(r.out[2]), r.ld[2], row0, col0, r.m, r.n);
                    }
                    gate(p.act, g, u);
                    store_block<T>(stage, g, static_cast<T*>(r.out[0]), r.ld[0], row0, col0, r.m, r.n);
                }
            } else {
                for (unsigned c = side * (kTile / 2); c < (side + 1) * (kTile / 2); c += 32) {
                    float v[32];
                    tc::load_columns(from + c, v);
                    if constexpr (kScaled)
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] *= unscale;
                    const unsigned col0 = t.col * kTile + c;
                    if (!t.paired && p.parts > 1) {   // this lane's row of a part, as it is
                        float* to = p.sums + ((size_t)t.part * r.m + row0 + lane) * p.sums_ld + col0;
                        if (row0 + lane < r.m)
#pragma unroll
                            for (int j = 0; j < 32; j += 4)
                                if (col0 + j < p.sums_ld) *reinterpret_cast<float4*>(to + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        __syncwarp();   // the next columns are read by the warp as one
                        continue;
                    }
                    store_block<T>(stage, v, static_cast<T*>(r.out[t.pair]), r.ld[t.pair], row0, col0, r.m, r.n);
                }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::barrier_arrive_in(tc::address_in(taken + 8 * acc, 0));
        }
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (*dead) tc::pause();   // a wait ran out: what is in flight between the two blocks lands before either ends
    tc::cluster_barrier();
    if (warp == 2) {
        tc::fence_after_sync();
        tc::tmem_free_pair(tmem, 2 * kTile);
    }
}

// ---- few tokens -----------------------------------------------------------------------------------------------------------------
//
// Bound by the one read of both weights.  The weights are the 128-row operand here (128 columns of each to a tile) and the tokens the
// narrow one, so that a slice in flight is nearly all weights.  The slices of all tiles, in order, are dealt out evenly: one
// block per SM takes a run of them, whole tiles or parts of tiles, through one ring that never drains, and leaves the sums of each
// (part of a) tile in the workspace; glu_few_finish_kernel adds the parts of a tile, in order, and applies the activation.
// Measured: one token through 4096 x 11008 bf16, 34 us with both kernels (5.3 TB/s of 6.56; reading the same boxes and nothing else 29 us); 48
// tokens through 5120 x 13824 f16, 55 to 57 us (5.1 TB/s).
// Parts of a cluster that share a tile through distributed shared memory were measured before: no more than one such block ran on an
// SM, and the ring of 72 KB that left to each read 4.0 TB/s.
constexpr int kFewCols = 128, kFewThreads = 256;
template <int kTokens> constexpr int kFewSlice = (2 * kFewCols + kTokens) * kDepth * 2;
template <int kTokens> constexpr int kFewRing = kTokens <= 32 ? 6 : kTokens == 64 ? 5 : 4;
template <int kTokens> constexpr size_t few_smem() { return 1024 + (size_t)kFewRing<kTokens> * kFewSlice<kTokens> + 256; }

struct FewArgs {
    CUtensorMap x, w[2];
    unsigned tokens, tiles, slices;   // slices: of a tile
    float* parts;                     // [tile + block][token][gate, up][128]
    int* flag;
};
struct FewEnd {
    const float* parts;
    unsigned tokens, hidden, tiles, slices, blocks;
    void* out[3];
    size_t ld[3];
    int act;
};
// the first slice of a block's run
__host__ __device__ __forceinline__ unsigned run_start(unsigned block, unsigned blocks, unsigned total) {
    return (unsigned)((unsigned long long)total * block / blocks);
}
// the block whose run holds a slice
__device__ __forceinline__ unsigned run_of(unsigned slice, unsigned blocks, unsigned total) {
    return (unsigned)((((unsigned long long)slice + 1) * blocks - 1) / total);
}

template <class T, int kTokens>
__global__ void __launch_bounds__(kFewThreads) glu_few_kernel(const __grid_constant__ FewArgs p) {
    constexpr int kA = kFewCols * kDepth * 2, kSlice = kFewSlice<kTokens>, kR = kFewRing<kTokens>;
    constexpr uint32_t kInstruction = tc::instruction<T>(kFewCols, kTokens, true, false);
    constexpr uint32_t kAcc = 2 * kTokens;
    extern __shared__ char raw[];
    char* ring = raw + ((1024 - (tc::smem_address(raw) & 1023)) & 1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kR * kSlice);
    volatile int* dead = reinterpret_cast<volatile int*>(bars + 2 * kR + 5);
    const uint32_t full = tc::smem_address(bars), empty = full + 8 * kR, ready = empty + 8 * kR, taken = ready + 16, drained = taken + 16;
    const uint32_t tmem_at = drained + 16;
    const tc::Watch watch = {dead, p.flag};
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned total = p.tiles * p.slices, first = run_start(blockIdx.x, gridDim.x, total), last = run_start(blockIdx.x + 1, gridDim.x, total);
    const auto fetch = [&](unsigned i) {   // the i-th slice of the run
        const unsigned s = first + i, at = i % kR, col = s / p.slices * kFewCols, k = s % p.slices * kDepth;
        const uint32_t a = tc::smem_address(ring) + at * kSlice, bar = full + 8 * at;
        tc::barrier_expect(bar, kSlice);
        for (int j = 0; j < kFewCols / 64; ++j) tc::load_box(&p.w[0], a + j * 8192, bar, col + j * 64, k);
        for (int j = 0; j < kFewCols / 64; ++j) tc::load_box(&p.w[1], a + kA + j * 8192, bar, col + j * 64, k);
        tc::load_box(&p.x, a + 2 * kA, bar, k, 0);
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < kR; ++i) {
            tc::barrier_init(full + 8 * i, 1);
            tc::barrier_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::barrier_init(ready + 8 * i, 1);
            tc::barrier_init(taken + 8 * i, 4);
        }
        tc::barrier_init(drained, 1);
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        grid_wait();
        for (unsigned i = 0; i < kR && first + i < last; ++i) fetch(i);   // the first copies need nothing else of what is set up here
    }
    if (warp == 2) tc::tmem_alloc(tmem_at, 2 * kAcc);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(bars + 2 * kR + 6);
    grid_release();
    grid_wait();

    if (warp == 0 && lane == 0) {
        unsigned issued = min((unsigned)kR, last - first);
        bool fine = true;
        for (; first + issued < last; ++issued) {
            if (!tc::barrier_wait(empty + 8 * (issued % kR), ((issued / kR) & 1) ^ 1, watch)) { fine = false; break; }
            fetch(issued);
        }
        if (!fine)
            for (unsigned i = issued > kR ? issued - kR : 0; i < issued; ++i) tc::barrier_wait(full + 8 * (i % kR), (i / kR) & 1, watch, true);
    } else if (warp == 1 && lane == 0) {
        unsigned used = 0, count = 0;
        bool fine = true;
        for (unsigned s = first; s < last; ++s, ++used) {
            const unsigned at = used % kR, acc = count & 1;
            const bool begin = s == first || s % p.slices == 0;
            if (begin && !tc::barrier_wait(taken + 8 * acc, ((count >> 1) & 1) ^ 1, watch)) { fine = false; break; }
            if (!tc::barrier_wait(full + 8 * at, (used / kR) & 1, watch)) { fine = false; break; }
            tc::fence_after_sync();
            const uint32_t a = tc::smem_address(ring) + at * kSlice, b = a + 2 * kA, d = tmem + acc * kAcc;
#pragma unroll
            for (int k = 0; k < kDepth / 16; ++k) {
                const uint64_t x = tc::tile_descriptor(b + k * 32, false, 0);
                tc::product(d, tc::tile_descriptor(a + k * 2048, true, 8192), x, kInstruction, !begin || k);
                tc::product(d + kTokens, tc::tile_descriptor(a + kA + k * 2048, true, 8192), x, kInstruction, !begin || k);
            }
            tc::commit(empty + 8 * at);
            if (s + 1 == last || (s + 1) % p.slices == 0) {
                tc::commit(ready + 8 * acc);
                ++count;
            }
        }
        if (!fine) {
            tc::commit(drained);
            tc::barrier_wait(drained, 0, watch, true);
        }
    } else if (warp >= 4 && first < last) {
        unsigned count = 0;
        for (unsigned tile = first / p.slices; tile <= (last - 1) / p.slices; ++tile, ++count) {
            const unsigned acc = count & 1;
            if (!tc::barrier_wait_warp(ready + 8 * acc, (count >> 1) & 1, watch)) break;
            tc::fence_after_sync();
            float* to = p.parts + (size_t)(tile + blockIdx.x) * p.tokens * 2 * kFewCols + (warp - 4) * 32 + lane;
            for (unsigned t0 = 0; t0 < p.tokens; t0 += 16) {
                float g[16], u[16];
                tc::load_columns16(tmem + ((warp - 4) * 32 << 16) + acc * kAcc + t0, g);
                tc::load_columns16(tmem + ((warp - 4) * 32 << 16) + acc * kAcc + kTokens + t0, u);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (t0 + i >= p.tokens) break;
                    to[(t0 + i) * 2 * kFewCols] = g[i];
                    to[(t0 + i) * 2 * kFewCols + kFewCols] = u[i];
                }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::barrier_arrive(taken + 8 * acc);
        }
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    // A wait ran out: where the copies were all issued before, or the products, nobody above has waited for them; they land before the block ends.
    if (*dead) tc::pause();
    if (warp == 2) {
        tc::fence_after_sync();
        tc::tmem_free(tmem, 2 * kAcc);
    }
}

// One block to 128 columns and kFewTogether tokens, whose parts are read together: four where there are more than that many tokens (48
// tokens: 1 us less than one by one), else one (a single token: 0.2 us less than as one of four).  Its blocks are launched while
// glu_few_kernel still runs and wait for its end.
template <class T, unsigned kFewTogether>
__global__ void __launch_bounds__(kFewCols) glu_few_finish_kernel(const __grid_constant__ FewEnd p) {
    const unsigned tile = blockIdx.x, t0 = blockIdx.y * kFewTogether, f = tile * kFewCols + threadIdx.x, total = p.tiles * p.slices;
    grid_release();
    grid_wait();
    const unsigned b0 = run_of(tile * p.slices, p.blocks, total), b1 = run_of(tile * p.slices + p.slices - 1, p.blocks, total);
    if (f >= p.hidden) return;
    float g[kFewTogether] = {}, u[kFewTogether] = {};
    for (unsigned b = b0; b <= b1; ++b) {
        const float* from = p.parts + ((size_t)(tile + b) * p.tokens + t0) * 2 * kFewCols + threadIdx.x;
#pragma unroll
        for (unsigned i = 0; i < kFewTogether; ++i)
            if (t0 + i < p.tokens) {
                g[i] += from[i * 2 * kFewCols];
                u[i] += from[i * 2 * kFewCols + kFewCols];
            }
    }
    float h[kFewTogether];
#pragma unroll
    for (unsigned i = 0; i < kFewTogether; ++i) h[i] = g[i];
    gate(p.act, h, u);
#pragma unroll
    for (unsigned i = 0; i < kFewTogether; ++i) {
        const unsigned t = t0 + i;
        if (t >= p.tokens) break;
        if (p.out[1]) {
            static_cast<T*>(p.out[1])[t * p.ld[1] + f] = from_f32<T>(g[i]);
            static_cast<T*>(p.out[2])[t * p.ld[2] + f] = from_f32<T>(u[i]);
        }
        static_cast<T*>(p.out[0])[t * p.ld[0] + f] = from_f32<T>(h[i]);
    }
}

// 8 values from any address, of which `count` (1 to 8) belong to the row; the others come back as they may.  Reads whole 16-byte
// granules, the second only where it holds one of the row's values, so that nothing beyond the row's own pages is touched.
template <class T>
__device__ __forceinline__ Vec<T, 8> load_any(const T* p, unsigned count) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const unsigned off = at & 15;
    const uint4* from = reinterpret_cast<const uint4*>(at - off);
    const uint4 a = __ldg(from);
    uint4 b = make_uint4(0, 0, 0, 0);
    if (off + count * 2 > 16) b = __ldg(from + 1);
    const uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const unsigned word = off >> 2, bits = (off & 3) * 8;
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = word < 2 ? (word ? x[i + 1] : x[i]) : (word == 2 ? x[i + 2] : x[i + 3]);
    union { uint32_t u[4]; Vec<T, 8> v; } out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out.u[i] = __funnelshift_r(w[i], w[i + 1], bits);
    return out.v;
}

// The gradients of the two projections' results.  They are rounded to the tensors' type, as the operands of the products that
// follow have to be: each is off by half a step at most, independently, so a sum over them is off by no more, relative to its
// norm, than its own rounding.  bf16 has the range of the 32 bits that they are formed in.  f16 has not - gradients of 1e-6 would keep a
// few bits, products above 65504 none - so there they are rounded at a scale, a power of two for the whole call that puts the largest of
// them at 2^14 to 2^15, and the products' 32-bit sums are scaled back: a gradient is off by 2^-39 of the largest at most where
// that is more than half its step (below 2^-29 of the largest).  The largest takes a pass of its own over the three inputs:
// 42 us for 2048 x 11008, as long as the rounding pass, of 650 us for the whole call; 12 us for 777 x 2731 in unaligned rows.
struct SplitArgs {
    const void *gate, *up, *dh;
    void *dg, *du;
    size_t ldg, ldu, ldh, ld;
    unsigned rows, cols;   // no rows: nothing to split
    int act;
    bool wide;
    float *peaks, *unscale;   // f16: the largest value that each of n_peaks blocks has seen; where the scale's inverse goes
    unsigned n_peaks;
};
// 8 values of both gradients from column n of row m on
template <class T>
__device__ __forceinline__ void split_values(const SplitArgs& a, unsigned m, unsigned n, float (&g)[8], float (&u)[8]) {
    const T *gate = static_cast<const T*>(a.gate) + m * a.ldg + n, *up = static_cast<const T*>(a.up) + m * a.ldu + n,
            *dh = static_cast<const T*>(a.dh) + m * a.ldh + n;
    float d[8];
    if (a.wide && n + 8 <= a.cols) {
        load_vec<T, 8>(gate, g);
        load_vec<T, 8>(up, u);
        load_vec<T, 8>(dh, d);
    } else {
        const unsigned count = min(8u, a.cols - n);
        const Vec<T, 8> x = load_any<T>(gate, count), y = load_any<T>(up, count), z = load_any<T>(dh, count);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = to_f32<T>(x.v[j]), u[j] = to_f32<T>(y.v[j]), d[j] = to_f32<T>(z.v[j]);
    }
    ungate(a.act, g, u, d);
}
// The largest of the values, none below zero, that the block's 128 threads hold; for every thread.
__device__ __forceinline__ float block_peak(float peak) {
    __shared__ unsigned part[4];
    const unsigned most = __reduce_max_sync(0xffffffffu, __float_as_uint(peak));   // floats without a sign are ordered like their bits
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = most;
    __syncthreads();
    return __uint_as_float(max(max(part[0], part[1]), max(part[2], part[3])));
}
// Infinities and NaN have no part in the scale: they stay what they are under any.
template <class T>
__global__ void __launch_bounds__(128) glu_peak_kernel(const __grid_constant__ SplitArgs a) {
    const unsigned n = (blockIdx.x * 128 + threadIdx.x) * 8;
    float peak = 0.0f;
    if (n < a.cols)
        for (unsigned m = blockIdx.y; m < a.rows; m += gridDim.y) {
            float g[8], u[8];
            split_values<T>(a, m, n, g, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = fabsf(g[j]), y = fabsf(u[j]);
                if (n + j < a.cols) peak = fmaxf(peak, fmaxf(isfinite(x) ? x : 0.0f, isfinite(y) ? y : 0.0f));
            }
        }
    peak = block_peak(peak);
    if (threadIdx.x == 0) a.peaks[blockIdx.y * gridDim.x + blockIdx.x] = peak;
}
template <class T>
__device__ __forceinline__ void split_rows(const SplitArgs& a) {
    float scale = 1.0f;
    if constexpr (std::is_same<T, __half>::value) {
        float peak = 0.0f;
        for (unsigned i = threadIdx.x; i < a.n_peaks; i += 128) peak = fmaxf(peak, a.peaks[i]);
        // 14 less the peak's exponent, -20 at least for products of f16 values; past 2^100 every result is zero in f16 anyway
        const int up = min(100, 14 + 127 - (int)(__float_as_uint(block_peak(peak)) >> 23));
        scale = __uint_as_float((unsigned)(127 + up) << 23);
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.unscale = __uint_as_float((unsigned)(127 - up) << 23);
    }
    const unsigned n = (blockIdx.x * 128 + threadIdx.x) * 8;
    if (n >= a.cols) return;
    for (unsigned m = blockIdx.y; m < a.rows; m += gridDim.y) {
        float g[8], u[8];
        split_values<T>(a, m, n, g, u);
        if constexpr (std::is_same<T, __half>::value)
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] *= scale, u[j] *= scale;
        store_vec<T, 8>(static_cast<T*>(a.dg) + m * a.ld + n, g);
        store_vec<T, 8>(static_cast<T*>(a.du) + m * a.ld + n, u);
    }
}

// dx from the parts of its sums, in their order
struct AddArgs {
    const float* sums;
    void* out;
    size_t ldo;
    unsigned parts, m, n, ld;   // no parts: nothing to add
    bool wide;
};
template <class T>
__device__ __forceinline__ void add_rows(const AddArgs& a) {
    const unsigned c = (blockIdx.x * 128 + threadIdx.x) * 4;
    if (c >= a.n) return;
    for (unsigned row = blockIdx.y; row < a.m; row += gridDim.y) {
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (unsigned k = 0; k < a.parts; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(a.sums + ((size_t)k * a.m + row) * a.ld + c);
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        const float v[4] = {s.x, s.y, s.z, s.w};
        T* to = static_cast<T*>(a.out) + (size_t)row * a.ldo + c;
        if (a.wide && c + 4 <= a.n) {
            store_vec<T, 4>(to, v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < a.n) to[j] = from_f32<T>(v[j]);
        }
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

// Rows that a tensor copy cannot read (an address or a stride that is no multiple of 16 bytes), laid out anew with a stride of
// whole 16 bytes: one pass over the operands before the products.
struct Operand { const void* p; size_t ld, rows, cols; };
struct AlignArgs {
    Operand from[3];
    void* to[3];
    size_t ld_to[3];
};
// What comes before the products, in one launch: the gradients of the projections (blockIdx.z 0, if asked for) and the operands.
template <class T>
__global__ void __launch_bounds__(128) glu_before_kernel(const __grid_constant__ SplitArgs split, const __grid_constant__ AlignArgs a) {
    unsigned z = blockIdx.z;
    if (split.rows) {
        if (z == 0) {
            split_rows<T>(split);
            return;
        }
        --z;
    }
    const Operand& x = a.from[z];
    const size_t c = (blockIdx.x * 128 + threadIdx.x) * 8, ld = a.ld_to[z];
    if (c >= ld) return;
    for (size_t r = blockIdx.y; r < x.rows; r += gridDim.y) {
        const Vec<T, 8> v = load_any<T>(static_cast<const T*>(x.p) + r * x.ld + c, (unsigned)min((size_t)8, x.cols - c));
        *reinterpret_cast<Vec<T, 8>*>(static_cast<T*>(a.to[z]) + r * ld + c) = v;
    }
}

// Results for addresses that take no 16-byte stores are formed in the workspace and brought to their places by 16-byte granules of
// the place; a row's first and last are written by value.
struct PlaceArgs {
    const void* from[3];
    void* to[3];
    size_t ld_from[3], ld_to[3];
    unsigned rows[3], cols[3], n;
};
template <class T>
__global__ void __launch_bounds__(128) glu_after_kernel(const __grid_constant__ PlaceArgs a, const __grid_constant__ AddArgs add) {
    const unsigned z = blockIdx.z;
    if (z == a.n) {
        add_rows<T>(add);
        return;
    }
    const int g = blockIdx.x * 128 + threadIdx.x, cols = (int)a.cols[z];
    for (size_t r = blockIdx.y; r < a.rows[z]; r += gridDim.y) {
        const T* from = static_cast<const T*>(a.from[z]) + r * a.ld_from[z];
        T* to = static_cast<T*>(a.to[z]) + r * a.ld_to[z];
        const int e = g * 8 - (int)((reinterpret_cast<uintptr_t>(to) & 15) / 2);   // the granule's first value
        if (e >= cols) continue;
        if (e >= 0 && e + 8 <= cols) {
            *reinterpret_cast<Vec<T, 8>*>(to + e) = load_any<T>(from + e, 8);
        } else {
            for (int j = max(e, 0); j < min(e + 8, cols); ++j) to[j] = from[j];
        }
    }
}

bool copyable(const void* p, size_t ld) { return aligned_to(p, 16) && ld % 8 == 0; }
// rows of a grid whose blocks take several each: as many as are resident at once (16 blocks of 128 threads to an SM), no more
unsigned grid_rows(size_t rows, unsigned blocks_a_row) { return (unsigned)std::min<size_t>(rows, std::max(1u, 16u * sm_count() / blocks_a_row)); }
// Makes operands readable by tensor copies, those that are not through the workspace, and splits the gradient where that is asked for.
template <class T>
int before(const SplitArgs& split, std::initializer_list<Operand*> operands, Scratch* scratch, cudaStream_t s) {
    AlignArgs a = {};
    unsigned n = 0, across = split.rows ? div_up(split.cols, 8 * 128) : 0;
    size_t rows = split.rows;
    for (Operand* x : operands) {
        const size_t ld = (x->cols + 7) / 8 * 8;
        if (x->rows == 1) x->ld = ld;   // never used
        if (copyable(x->p, x->ld)) continue;
        a.from[n] = *x;
        a.ld_to[n] = ld;
        if (!(a.to[n] = scratch->get_n<T>(x->rows * ld))) return ZKB_ERR_CUDA;
        x->p = a.to[n], x->ld = ld;
        rows = std::max(rows, x->rows), across = std::max(across, div_up(ld, 8 * 128));
        ++n;
    }
    n += split.rows != 0;
    if (!n) return ZKB_OK;
    const auto glu_before = glu_before_kernel<T>;
    ZKB_LAUNCH(glu_before, dim3(across, grid_rows(rows, across * n), n), 128, 0, s, split, a);
    return ZKB_OK;
}

template <class T, class Args>
int product_launch(const Args& p, size_t tiles, cudaStream_t s) {
    const auto glu_product = glu_product_kernel<T, Args>;
    ZKB_CUDA(cudaFuncSetAttribute(glu_product, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kProductSmem));
    // A plain launch, and no trigger in the kernel.  While it took part in programmatic launches, a loop of gradient calls stalled twice; the
    // cause is open (a successor starts only when every block has triggered, so it cannot have taken a cluster's place, and the warps that
    // could part before instructions on tensor memory were mended at the same time), so it stays out of them.
    ZKB_LAUNCH(glu_product, 2 * (unsigned)std::min(tiles, (size_t)sm_count() / 2), kProductThreads, kProductSmem, s, p);
    return ZKB_OK;
}
void lay_results(Results* r, size_t m, size_t n, unsigned tile_cols, size_t k) {
    r->m = (unsigned)m, r->n = (unsigned)n, r->slices = div_up(k, kDepth);
    r->row_tiles = div_up(m, kTile), r->col_tiles = div_up(n, tile_cols);
}
// Sets a result's place, or room for it in the workspace and a note of where it goes.
template <class T>
int set_result(Results* r, int i, void* out, size_t ld, Scratch* scratch, PlaceArgs* later) {
    r->out[i] = out, r->ld[i] = ld;
    if (!out || copyable(out, ld)) return ZKB_OK;
    r->ld[i] = (r->n + 7) / 8 * 8;
    if (!(r->out[i] = scratch->get_n<T>((size_t)r->m * r->ld[i]))) return ZKB_ERR_CUDA;
    const unsigned n = later->n++;
    later->from[n] = r->out[i], later->ld_from[n] = r->ld[i];
    later->to[n] = out, later->ld_to[n] = ld;
    later->rows[n] = r->m, later->cols[n] = r->n;
    return ZKB_OK;
}
template <class T>
int after(const PlaceArgs& a, const AddArgs& add, cudaStream_t s) {
    unsigned across = add.parts ? div_up(add.n, 4 * 128) : 0, rows = add.parts ? add.m : 0;
    for (unsigned i = 0; i < a.n; ++i) across = std::max(across, div_up(a.cols[i] + 7, 8 * 128)), rows = std::max(rows, a.rows[i]);
    const unsigned n = a.n + (add.parts != 0);
    if (!n) return ZKB_OK;
    const auto glu_after = glu_after_kernel<T>;
    ZKB_LAUNCH(glu_after, dim3(across, grid_rows(rows, across * n), n), 128, 0, s, a, add);
    return ZKB_OK;
}

template <class T> constexpr int kCode = std::is_same<T, __half>::value ? ZKB_F16 : ZKB_BF16;

template <class T, int kTokens>
int glu_few_launch(const GluArgs& a, Operand x, Operand wg, Operand wu, int* flag, Scratch* scratch, cudaStream_t s) {
    FewArgs p = {};
    ZKB_TRY(tc::make_map(&p.x, kCode<T>, x.p, a.tokens, a.in, x.ld, kTokens));
    ZKB_TRY(tc::make_map(&p.w[0], kCode<T>, wg.p, a.in, a.hidden, wg.ld, kDepth));
    ZKB_TRY(tc::make_map(&p.w[1], kCode<T>, wu.p, a.in, a.hidden, wu.ld, kDepth));
    p.tokens = (unsigned)a.tokens, p.tiles = div_up(a.hidden, kFewCols), p.slices = div_up(a.in, kDepth), p.flag = flag;
    const unsigned blocks = (unsigned)std::min((size_t)sm_count(), (size_t)p.tiles * p.slices);
    p.parts = scratch->get_n<float>((size_t)(p.tiles + blocks) * p.tokens * 2 * kFewCols);
    if (!p.parts) return ZKB_ERR_CUDA;
    const auto glu_few = glu_few_kernel<T, kTokens>;
    constexpr size_t smem = few_smem<kTokens>();
    ZKB_CUDA(cudaFuncSetAttribute(glu_few, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    ZKB_TRY(launch_beside("glu_few", glu_few, blocks, kFewThreads, smem, s, p));
    const FewEnd e = {p.parts, p.tokens, (unsigned)a.hidden, p.tiles, p.slices, blocks, {a.h, a.gate_out, a.up_out}, {a.ldh, a.ldg, a.ldu}, a.act};
    const unsigned together = p.tokens > 4 ? 4 : 1;
    const auto glu_few_finish = together == 4 ? glu_few_finish_kernel<T, 4> : glu_few_finish_kernel<T, 1>;
    return launch_beside("glu_few_finish", glu_few_finish, dim3(p.tiles, div_up(p.tokens, together)), kFewCols, 0, s, e);
}

template <class T>
int glu_launch(const GluArgs& a, cudaStream_t s) {
    if (!a.in) {   // a sum over nothing
        for (auto [p, ld] : {std::pair<void*, size_t>{a.h, a.ldh}, {a.gate_out, a.ldg}, {a.up_out, a.ldu}})
            if (p) ZKB_CUDA(cudaMemset2DAsync(p, ld * 2, 0, a.hidden * 2, a.tokens, s));
        return ZKB_OK;
    }
    Scratch scratch(s);
    Operand x = {a.x, a.ldx, a.tokens, a.in}, wg = {a.wg, a.ldwg, a.in, a.hidden}, wu = {a.wu, a.ldwu, a.in, a.hidden};
    ZKB_TRY(before<T>(SplitArgs{}, {&x, &wg, &wu}, &scratch, s));
    int* const flag = tc::wait_flag();
    if (!flag) return ZKB_ERR_CUDA;
    // The border: 4096 x 11008 bf16 takes 37 us for 16 tokens, 38 for 32, 41 for 64 and 44.5 for 128 with the tokens as the narrow operand, and
    // 53 us for 129 as for 256 in the product kernel, whose tiles are 256 tokens high whatever they hold.
    if (a.tokens <= 16) return glu_few_launch<T, 16>(a, x, wg, wu, flag, &scratch, s);
    if (a.tokens <= 32) return glu_few_launch<T, 32>(a, x, wg, wu, flag, &scratch, s);
    if (a.tokens <= 64) return glu_few_launch<T, 64>(a, x, wg, wu, flag, &scratch, s);
    if (a.tokens <= 128) return glu_few_launch<T, 128>(a, x, wg, wu, flag, &scratch, s);
    GatedArgs p = {};
    p.act = a.act, p.flag = flag;
    ZKB_TRY(tc::make_map(&p.a, kCode<T>, x.p, a.tokens, a.in, x.ld, kHalf));
    ZKB_TRY(tc::make_map(&p.b[0], kCode<T>, wg.p, a.in, a.hidden, wg.ld, kDepth));
    ZKB_TRY(tc::make_map(&p.b[1], kCode<T>, wu.p, a.in, a.hidden, wu.ld, kDepth));
    lay_results(&p.r, a.tokens, a.hidden, kHalf, a.in);
    PlaceArgs later = {};
    ZKB_TRY(set_result<T>(&p.r, 0, a.h, a.ldh, &scratch, &later));
    ZKB_TRY(set_result<T>(&p.r, 1, a.gate_out, a.ldg, &scratch, &later));
    ZKB_TRY(set_result<T>(&p.r, 2, a.up_out, a.ldu, &scratch, &later));
    ZKB_TRY(product_launch<T>(p, (size_t)p.r.row_tiles * p.r.col_tiles, s));
    return after<T>(later, AddArgs{}, s);
}

template <class T>
int glu_backward_launch(const GluArgs& a, cudaStream_t s) {
    const size_t F = a.hidden, ld = (F + 7) / 8 * 8;
    if (!F || !a.tokens) {   // sums over nothing
        if (a.dx && a.tokens) ZKB_CUDA(cudaMemset2DAsync(a.dx, a.lddx * 2, 0, a.in * 2, a.tokens, s));
        if (a.dwg && F) ZKB_CUDA(cudaMemset2DAsync(a.dwg, a.lddwg * 2, 0, F * 2, a.in, s));
        if (a.dwu && F) ZKB_CUDA(cudaMemset2DAsync(a.dwu, a.lddwu * 2, 0, F * 2, a.in, s));
        return ZKB_OK;
    }
    if (!a.dx && !a.dwg) return ZKB_OK;
    Scratch scratch(s);
    const dim3 peak_grid(div_up(F, 8 * 128), grid_rows(a.tokens, 2 * div_up(F, 8 * 128)));   // 8 blocks to an SM: fewer peaks to read again
    const unsigned n_peaks = std::is_same<T, __half>::value ? peak_grid.x * peak_grid.y : 0;
    T* const dg = scratch.get_n<T>(2 * a.tokens * ld + (n_peaks + 1) * sizeof(float) / sizeof(T));
    if (!dg) return ZKB_ERR_CUDA;
    T* const du = dg + a.tokens * ld;
    float* const peaks = reinterpret_cast<float*>(du + a.tokens * ld);   // rows are whole 16 bytes
    const SplitArgs split = {a.gate, a.up, a.dh, dg, du, a.ldg, a.ldu, a.lddh, ld, (unsigned)a.tokens, (unsigned)F, a.act,
                             copyable(a.gate, a.ldg) && copyable(a.up, a.ldu) && copyable(a.dh, a.lddh), peaks, peaks + n_peaks, n_peaks};
    if constexpr (std::is_same<T, __half>::value) {
        const auto glu_peak = glu_peak_kernel<T>;
        ZKB_LAUNCH(glu_peak, peak_grid, 128, 0, s, split);
    }
    Operand x = {a.x, a.ldx, a.tokens, a.in}, wg = {a.wg, a.ldwg, a.in, F}, wu = {a.wu, a.ldwu, a.in, F};
    if (a.dx && a.dwg) ZKB_TRY(before<T>(split, {&x, &wg, &wu}, &scratch, s));
    else if (a.dx) ZKB_TRY(before<T>(split, {&wg, &wu}, &scratch, s));
    else ZKB_TRY(before<T>(split, {&x}, &scratch, s));
    GradArgs p = {};
    p.unscale = split.unscale;
    PlaceArgs later = {};
    AddArgs add = {};
    if (!(p.flag = tc::wait_flag())) return ZKB_ERR_CUDA;
    if (a.dx) {
        ZKB_TRY(tc::make_map(&p.dg_rows[0], kCode<T>, dg, a.tokens, F, ld, kHalf));
        ZKB_TRY(tc::make_map(&p.dg_rows[1], kCode<T>, du, a.tokens, F, ld, kHalf));
        ZKB_TRY(tc::make_map(&p.w[0], kCode<T>, wg.p, a.in, F, wg.ld, kHalf));
        ZKB_TRY(tc::make_map(&p.w[1], kCode<T>, wu.p, a.in, F, wu.ld, kHalf));
        lay_results(&p.dx, a.tokens, a.in, kTile, F);
    }
    if (a.dwg) {
        ZKB_TRY(tc::make_map(&p.x, kCode<T>, x.p, a.tokens, a.in, x.ld, kDepth));
        ZKB_TRY(tc::make_map(&p.dg_cols[0], kCode<T>, dg, a.tokens, F, ld, kDepth));
        ZKB_TRY(tc::make_map(&p.dg_cols[1], kCode<T>, du, a.tokens, F, ld, kDepth));
        lay_results(&p.dw, a.in, F, kTile, a.tokens);
        ZKB_TRY(set_result<T>(&p.dw, 0, a.dwg, a.lddwg, &scratch, &later));
        ZKB_TRY(set_result<T>(&p.dw, 1, a.dwu, a.lddwu, &scratch, &later));
    }
    // at least 8 slices to a part: fewer cost more in the sums' way through memory than they save
    const size_t whole = (size_t)p.dx.row_tiles * p.dx.col_tiles, most = sm_count() / 2;
    p.parts = whole && whole < most ? (unsigned)std::max<size_t>(1, std::min<size_t>(most / whole, 2 * p.dx.slices / 8)) : 1;
    if (p.parts > 1) {
        p.sums_ld = (p.dx.n + 3) / 4 * 4;
        p.sums = scratch.get_n<float>((size_t)p.parts * p.dx.m * p.sums_ld);
        if (!p.sums) return ZKB_ERR_CUDA;
        add = {p.sums, a.dx, a.lddx, p.parts, p.dx.m, p.dx.n, p.sums_ld, copyable(a.dx, a.lddx)};
    } else if (a.dx) {
        ZKB_TRY(set_result<T>(&p.dx, 0, a.dx, a.lddx, &scratch, &later));
    }
    const size_t longs = whole * p.parts, shorts = 2 * (size_t)p.dw.row_tiles * p.dw.col_tiles;
    const size_t pairs = std::min(longs + shorts, most), spare = pairs - longs % pairs;
    // A tile costs its slices, but no less than the 16 slices' time that taking it out takes.
    const unsigned cost_long = std::max(16u, 2 * p.dx.slices / p.parts), cost_short = std::max(16u, p.dw.slices);
    if (shorts && longs % pairs) p.head = (unsigned)std::min<size_t>((cost_long + cost_short / 2) / cost_short, shorts / spare);
    ZKB_TRY(product_launch<T>(p, longs + shorts, s));
    return after<T>(later, add, s);
}

int check_matrix(const char* who, const char* name, const void* p, size_t rows, size_t cols, size_t ld, bool needed) {
    if (!p) return needed ? fail(ZKB_ERR_ARG, std::string(who) + ": " + name + " is missing") : ZKB_OK;
    if (ld < cols && rows > 1) return fail(ZKB_ERR_DIM, std::string(who) + ": " + name + ": row stride below the row's length");
    return check_device(p, 2, who, name);
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

namespace tc {

static std::atomic<int*> g_wait_flag{nullptr};

int* wait_flag() {
    static std::mutex mutex;
    if (int* made = g_wait_flag.load()) return made;
    std::lock_guard<std::mutex> lock(mutex);
    if (!g_wait_flag.load()) {
        const SetupDuringCapture setup;
        void* p = nullptr;
        const cudaError_t e = cudaHostAlloc(&p, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
        if (e != cudaSuccess) {
            cuda_fail(e, "cudaHostAlloc(wait flag)");
            return nullptr;
        }
        *static_cast<volatile int*>(p) = 0;
        g_wait_flag.store(static_cast<int*>(p));
    }
    return g_wait_flag.load();
}
int check_wait_flag(const char* who) {
    const volatile int* const f = g_wait_flag.load();
    if (!f || !*f) return ZKB_OK;
    return fail(ZKB_ERR_CUDA, std::string(who) + ": a wait of an earlier call of the float operators ran out, its results are incomplete (zkb_wait_status resets this)");
}

int make_map(CUtensorMap* map, int dtype, const void* p, size_t rows, size_t cols, size_t ld, unsigned box_rows) {
    static std::atomic<void*> entry{nullptr};
    void* fn = entry.load();
    if (!fn) {
        cudaDriverEntryPointQueryResult found;
        ZKB_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
        if (!fn || found != cudaDriverEntryPointSuccess) return fail(ZKB_ERR_CUDA, "tensor copies: the driver has no cuTensorMapEncodeTiled");
        entry.store(fn);
    }
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * 2};
    const cuuint32_t box[2] = {64, box_rows}, steps[2] = {1, 1};
    const CUresult e = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn)(
        map, dtype == ZKB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, box, steps,
        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (e != CUDA_SUCCESS) return fail(ZKB_ERR_CUDA, "cuTensorMapEncodeTiled: error " + std::to_string((int)e));
    return ZKB_OK;
}

}  // namespace tc
}  // namespace zkb

using namespace zkb;

extern "C" {

int zkb_wait_status(int reset) {
    const int rc = tc::check_wait_flag("zkb_wait_status");
    if (rc != ZKB_OK && reset) *static_cast<volatile int*>(tc::wait_flag()) = 0;
    return rc;
}

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
    ZKB_TRY(tc::check_wait_flag(who));
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
    ZKB_TRY(tc::check_wait_flag(who));
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
