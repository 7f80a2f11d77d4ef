// Rotary positions of queries and keys.
//
// Pair i of a head at position p is turned by the angle p * f_i:
//     (a, b) -> m (a cos - b sin, b cos + a sin),
// with (a, b) = (x[i], x[i + R/2]) in the half layout and (x[2i], x[2i + 1]) in the interleaved one; the other head_dim - R
// values of a head are copied.  The gradient is the same turn by the opposite angle.
#include <algorithm>

#include "floatops.cuh"

namespace zkb {
namespace {

constexpr int kMaxTensors = 4;
constexpr int kRopeThreads = 128;

struct RopeTensor {
    const void* in;
    void* out;
    long long ib, it, ih, ob, ot, oh;
    unsigned heads;
    bool copy_tail;        // out is not in: the values behind the turned ones have to be brought over
};
struct RopeArgs {
    RopeTensor t[kMaxTensors];
    unsigned n_tensors, heads /* the most of a tensor */, batch_tokens, tokens, half, tail, tokens_per_block;
    const double* inv_freq;
    float magnitude, sin_sign;
    const long long* positions;
    long long position_stride, first_position;
};

// Bound by HBM: each value is read and written once.  A block takes a few tokens: their sines and cosines are formed once,
// in shared memory, and serve every head of a tensor (blockIdx.z).  The angle is reduced to a fraction of a turn in 64 bits (a
// 32-bit product is off by 0.01 radians at position 131072) and only the fraction is rounded to 32.
// P pairs make a unit of work, in 16-byte vectors where sizes, strides and addresses allow it, else one pair at a time.  A thread
// keeps its unit and goes through the heads of the block's tokens, kAhead at a time so that their loads are in flight together.
// Measured: 3 x 4097 tokens, 48 heads of 128, f32, 100 us (6.0 TB/s of 6.56), 107 with the host's call; 2048 tokens, 64 heads, bf16, 18.5 us with the
// host's call.  Units dealt out anew for each vector (a division each) took 168 us for the first; four heads at a time needed 127
// registers and took 29 us for the second; 128 threads and 4 tokens to a block beat 256 and 8 by 2 us there.
template <class T, bool kWidePath, bool kInterleaved>
__global__ void __launch_bounds__(kRopeThreads, 8) rope_kernel(const __grid_constant__ RopeArgs a) {
    extern __shared__ float2 turn[];
    const RopeTensor& x = a.t[blockIdx.z];
    const unsigned tok0 = blockIdx.x * a.tokens_per_block;
    const unsigned n_tok = min(a.tokens_per_block, a.batch_tokens - tok0);
    for (unsigned i = threadIdx.x; i < n_tok * a.half; i += kRopeThreads) {
        const unsigned t = tok0 + i / a.half, b = t / a.tokens, s = t % a.tokens;
        const long long pos = a.positions ? a.positions[b * a.position_stride + s] : a.first_position + s;
        double turns = (double)pos * (a.inv_freq[i % a.half] * 0.15915494309189533577);
        turns -= rint(turns);
        float sn, cs;
        sincospif((float)(2.0 * turns), &sn, &cs);
        turn[i] = make_float2(cs * a.magnitude, sn * a.magnitude * a.sin_sign);
    }
    __syncthreads();

    constexpr int V = kWidePath ? kWide<T> : 1;
    constexpr int P = kWidePath && kInterleaved ? V / 2 : V;
    constexpr int N = kWidePath && !kInterleaved ? 2 : 1;   // vectors of a unit
    const unsigned turned = a.half / P;                     // P divides half
    const unsigned units = turned + a.tail / V;
    const unsigned side = min(units, (unsigned)kRopeThreads), lanes = kRopeThreads / side;   // threads to a head, heads at a time
    if (threadIdx.x >= side * lanes) return;
    const unsigned heads_here = (x.heads + gridDim.y - 1) / gridDim.y, head0 = blockIdx.y * heads_here;
    const unsigned n_heads = head0 < x.heads ? min(heads_here, x.heads - head0) : 0, rows = n_tok * n_heads;
    constexpr int kAhead = 2;
    for (unsigned u = threadIdx.x % side; u < units; u += side) {
        const bool copy = u >= turned;
        if (copy && !x.copy_tail) break;
        // where the unit's first and second values of its pairs begin
        const unsigned lo = copy ? 2 * a.half + (u - turned) * V : kInterleaved ? 2 * P * u : P * u;
        const unsigned hi = kInterleaved ? lo + 1 : a.half + lo;
        for (unsigned r0 = threadIdx.x / side; r0 < rows; r0 += kAhead * lanes) {
            Vec<T, V> v[kAhead][N];
            T second[kAhead], *to[kAhead];
            unsigned token[kAhead];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const unsigned r = r0 + q * lanes;
                to[q] = nullptr;
                if (r >= rows) continue;
                token[q] = r / n_heads;
                const unsigned h = head0 + r - token[q] * n_heads, t = tok0 + token[q], b = t / a.tokens, s = t - b * a.tokens;
                const T* in = static_cast<const T*>(x.in) + (b * x.ib + s * x.it + h * x.ih);
                to[q] = static_cast<T*>(x.out) + (b * x.ob + s * x.ot + h * x.oh);
                v[q][0] = *reinterpret_cast<const Vec<T, V>*>(in + lo);
                if constexpr (N == 2) {
                    if (!copy) v[q][1] = *reinterpret_cast<const Vec<T, V>*>(in + hi);
                }
                if constexpr (!kWidePath) {
                    if (!copy) second[q] = in[hi];
                }
            }
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                T* const out = to[q];
                if (!out) continue;
                if (copy) {
                    *reinterpret_cast<Vec<T, V>*>(out + lo) = v[q][0];
                    continue;
                }
                const float2* cs = turn + token[q] * a.half + u * P;
                Vec<T, V> w[N];
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const float2 c = cs[j];
                    const float x0 = to_f32<T>(kWidePath && kInterleaved ? v[q][0].v[2 * j] : v[q][0].v[j]);
                    const float x1 = to_f32<T>(!kWidePath ? second[q] : kInterleaved ? v[q][0].v[(2 * j + 1) % V] : v[q][N - 1].v[j]);
                    const T y0 = from_f32<T>(x0 * c.x - x1 * c.y), y1 = from_f32<T>(x1 * c.x + x0 * c.y);
                    if constexpr (kWidePath && kInterleaved) {
                        w[0].v[2 * j] = y0;
                        w[0].v[2 * j + 1] = y1;
                    } else {
                        w[0].v[j] = y0;
                        if constexpr (kWidePath) w[N - 1].v[j] = y1;
                        else out[hi] = y1;
                    }
                }
                *reinterpret_cast<Vec<T, V>*>(out + lo) = w[0];
                if constexpr (N == 2) *reinterpret_cast<Vec<T, V>*>(out + hi) = w[1];
            }
        }
    }
}

template <class T>
int rope_launch(RopeArgs a, bool interleaved, bool wide, cudaStream_t s) {
    a.tokens_per_block = a.half >= 512 ? 1 : std::min(4u, 512 / a.half);
    // few tokens: fewer to a block, then the heads over several blocks, until every SM has work
    const unsigned target = 2 * sm_count();
    while (a.tokens_per_block > 1 && div_up(a.batch_tokens, a.tokens_per_block) * a.n_tensors < target) a.tokens_per_block >>= 1;
    const unsigned gx = div_up(a.batch_tokens, a.tokens_per_block);
    const unsigned gy = gx * a.n_tensors >= target ? 1 : std::min(a.heads, target / (gx * a.n_tensors));
    const dim3 grid(gx, gy, a.n_tensors);
    const size_t smem = sizeof(float2) * a.tokens_per_block * a.half;
    const auto rope = interleaved ? (wide ? rope_kernel<T, true, true> : rope_kernel<T, false, true>)
                                  : (wide ? rope_kernel<T, true, false> : rope_kernel<T, false, false>);
    ZKB_LAUNCH(rope, grid, kRopeThreads, smem, s, a);
    return ZKB_OK;
}

}  // namespace

}  // namespace zkb

using namespace zkb;

extern "C" {

int zkb_rope_frequencies(int scaling, unsigned rotary_dim, double base, double factor, double original_len, double fast_turns, double slow_turns,
                         double* h_inv_freq, float* h_magnitude) {
    if (!h_inv_freq || !h_magnitude) return fail(ZKB_ERR_ARG, "zkb_rope_frequencies: no output");
    if (!rotary_dim || rotary_dim % 2) return fail(ZKB_ERR_DIM, "zkb_rope_frequencies: rotary_dim has to be even and positive");
    if (scaling < ZKB_ROPE_PLAIN || scaling > ZKB_ROPE_RAMP) return fail(ZKB_ERR_ARG, "zkb_rope_frequencies: unknown scaling");
    if (!(base > 1.0) || !std::isfinite(base)) return fail(ZKB_ERR_ARG, "zkb_rope_frequencies: base has to be above 1");
    if (scaling != ZKB_ROPE_PLAIN && !(factor >= 1.0 && std::isfinite(factor)))
        return fail(ZKB_ERR_ARG, "zkb_rope_frequencies: factor has to be 1 or more");
    const double n = rotary_dim;
    if (scaling == ZKB_ROPE_BASE && rotary_dim > 2) base *= std::pow(factor, n / (n - 2));
    double low = 0, high = 0;
    if (scaling == ZKB_ROPE_RAMP) {
        if (!(original_len > 0 && std::isfinite(original_len) && slow_turns > 0 && fast_turns > slow_turns && std::isfinite(fast_turns)))
            return fail(ZKB_ERR_ARG, "zkb_rope_frequencies: the ramp needs original_len > 0 and fast_turns > slow_turns > 0");
        // the pair that makes `turns` turns over the original context
        auto at = [&](double turns) { return n * std::log(original_len / (turns * 6.283185307179586477)) / (2 * std::log(base)); };
        low = std::max(std::floor(at(fast_turns)), 0.0);
        high = std::min(std::ceil(at(slow_turns)), n - 1);
    }
    for (unsigned i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / n);
        if (scaling == ZKB_ROPE_LINEAR) f /= factor;
        if (scaling == ZKB_ROPE_RAMP) {
            const double share = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
            f = f / factor * share + f * (1 - share);
        }
        h_inv_freq[i] = f;
    }
    *h_magnitude = scaling == ZKB_ROPE_RAMP ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return ZKB_OK;
}

int zkb_rope(int dtype, const zkb_rope_tensor_t* h_tensors, unsigned n_tensors, size_t batch, size_t tokens, size_t head_dim, size_t rotary_dim,
             int interleaved, const double* d_inv_freq, float magnitude, const int64_t* d_positions, int64_t position_batch_stride,
             int64_t first_position, int backward, void* stream) {
    ZKB_API_RANGE();
    if (!known_type(dtype)) return fail(ZKB_ERR_ARG, "zkb_rope: unknown type");
    if (n_tensors > kMaxTensors) return fail(ZKB_ERR_LIMIT, "zkb_rope: more than 4 tensors");
    if (n_tensors && !h_tensors) return fail(ZKB_ERR_ARG, "zkb_rope: no tensors");
    if (!rotary_dim || rotary_dim % 2 || rotary_dim > head_dim)
        return fail(ZKB_ERR_DIM, "zkb_rope: rotary_dim has to be even, positive and at most head_dim");
    if (head_dim > 8192) return fail(ZKB_ERR_LIMIT, "zkb_rope: head_dim above 8192");
    ZKB_TRY(tc::check_wait_flag("zkb_rope"));
    if (!n_tensors || !batch || !tokens) return ZKB_OK;
    if (tokens > 0x7fffffffull || batch > 0x7fffffffull || batch * tokens > 0x7fffffffull)
        return fail(ZKB_ERR_LIMIT, "zkb_rope: 2^31 tokens or more");
    if (!d_inv_freq) return fail(ZKB_ERR_ARG, "zkb_rope: no frequencies");
    ZKB_TRY(check_device(d_inv_freq, 8, "zkb_rope", "d_inv_freq"));
    ZKB_TRY(check_device(d_positions, 8, "zkb_rope", "d_positions"));

    RopeArgs a = {};
    const size_t es = type_size(dtype), v = 16 / es;
    bool wide = (rotary_dim / 2) % (interleaved ? v / 2 : v) == 0 && (head_dim - rotary_dim) % v == 0;
    for (unsigned k = 0; k < n_tensors; ++k) {
        const zkb_rope_tensor_t& h = h_tensors[k];
        if (!h.heads) continue;
        if (!h.d_in || !h.d_out) return fail(ZKB_ERR_ARG, "zkb_rope: tensor without memory");
        if (h.heads > 65535) return fail(ZKB_ERR_LIMIT, "zkb_rope: more than 65535 heads");
        ZKB_TRY(check_device(h.d_in, es, "zkb_rope", "d_in"));
        ZKB_TRY(check_device(h.d_out, es, "zkb_rope", "d_out"));
        const bool same = h.d_in == h.d_out;
        if (same && (h.in_batch != h.out_batch || h.in_token != h.out_token || h.in_head != h.out_head))
            return fail(ZKB_ERR_ARG, "zkb_rope: in place with other strides");
        for (unsigned j = 0; j < a.n_tensors; ++j)
            if (a.t[j].out == h.d_out) return fail(ZKB_ERR_ARG, "zkb_rope: two tensors with one output");
        RopeTensor& x = a.t[a.n_tensors++];
        x = {h.d_in, h.d_out, h.in_batch, h.in_token, h.in_head, h.out_batch, h.out_token, h.out_head, (unsigned)h.heads, !same};
        a.heads = std::max(a.heads, (unsigned)h.heads);
        const long long strides[6] = {x.ib, x.it, x.ih, x.ob, x.ot, x.oh};
        for (long long st : strides) wide = wide && st % (long long)v == 0;
        wide = wide && aligned_to(h.d_in, 16) && aligned_to(h.d_out, 16);
    }
    if (!a.n_tensors) return ZKB_OK;
    a.batch_tokens = (unsigned)(batch * tokens);
    a.tokens = (unsigned)tokens;
    a.half = (unsigned)(rotary_dim / 2);
    a.tail = (unsigned)(head_dim - rotary_dim);
    a.inv_freq = d_inv_freq;
    a.magnitude = magnitude;
    a.sin_sign = backward ? -1.0f : 1.0f;
    a.positions = reinterpret_cast<const long long*>(d_positions);
    a.position_stride = position_batch_stride;
    a.first_position = first_position;
    const cudaStream_t s = as_stream(stream);
    if (dtype == ZKB_F32) return rope_launch<float>(a, interleaved != 0, wide, s);
    if (dtype == ZKB_F16) return rope_launch<__half>(a, interleaved != 0, wide, s);
    return rope_launch<bf16>(a, interleaved != 0, wide, s);
}

}  // extern "C"
