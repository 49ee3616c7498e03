// Dropout between layers whose mask is never stored: whether element i (row-major) is kept is a function of i, a seed and a stream
// number, so the backward pass forms it again where it needs it.
//   words(q) = philox4x32_10(counter = (q low, q high, stream, "DROP"), key = seed),  keep(i) = words(i / 4)[i % 4] >= T,
//   T = round(p 2^32);   out[i] = keep(i) ? f(x[i]) / (1 - p) : 0,   f = identity or max(x, 0)
// One counter makes four elements, whatever their type, so that fp32 and bf16 rows of one seed lose the same elements; 32 bits an
// element, so that p is met to 2^-33.  The tag in the counter's last word keeps the sampler's streams of the same seed apart.
//
// With f = max(x, 0) the backward pass needs no generator: an element is kept and positive if and only if the output is not zero or
// below (it is no smaller than x, as 1 / (1 - p) >= 1), and the output is there for the next layer's own gradient anyway.
//
// What bounds it: the pass over memory.  60 K x 256 fp32, forward or backward: 21 us, 5.9 TB/s as the kernel sees it (what was written just before is
// read from the last-level cache); 2.4 M x 64 of rows of 100 columns: 277 us, back without gaps 202 us (6.1 TB/s).  In bf16 the generator's forty
// 32-bit products for four elements are as long: 87 K x 256 with relu 24.5 us forward, 20.7 us backward with 1.5 times the bytes and no generator.
#include "fgl_common.hpp"
#include "fgl_kernels.hpp"

#include <math.h>

namespace fgl {

constexpr uint32_t kDropTag = 0x44524F50u;
constexpr int kDropQuads = 4;  // fours of elements a thread: four loads on their way at once
constexpr int kDropTile = kBlock * kDropQuads * 4;
constexpr int64_t kDropMost = 1LL << 35;  // elements of a call: a launch has fewer than 2^32 threads

struct DropArgs {
    const void* x;
    void* out;
    int64_t n;       // elements
    int64_t ldx;     // of rows of n_cols elements (the kernel of flat arrays takes x as one row)
    uint32_t n_cols;
    uint32_t magic;  // ceil(2^32 / n_cols)
    uint32_t threshold;
    uint32_t stream_id;
    const int32_t* d_stream_offset;
    uint32_t seed_lo, seed_hi;
    float scale;
    int none;        // p = 1: nothing is kept
};

template <typename T>
struct DropType;
template <>
struct DropType<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct DropType<__bf16> {
    static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};

// A vector of four elements, aligned as one of them is.
template <typename T>
using DropQuad = T __attribute__((ext_vector_type(4), aligned(sizeof(T))));

template <bool RELU>
__device__ __forceinline__ float drop_value(float v, uint32_t word, const DropArgs& g)
{
    if constexpr (RELU) v = v <= 0.0f ? 0.0f : v;  // (what is not a number stays it)
    return word >= g.threshold && !g.none ? v * g.scale : 0.0f;
}

// FLAT: x is one array; else rows of n_cols elements at a distance of ldx, and out is one array all the same.
template <typename T, bool RELU, bool FLAT>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const DropArgs g)
{
    const T* x = static_cast<const T*>(g.x);
    T* out = static_cast<T*>(g.out);
    const int64_t tile0 = (int64_t)blockIdx.x * kDropTile;
    const uint32_t stream_id = g.stream_id + (g.d_stream_offset != nullptr ? (uint32_t)*g.d_stream_offset : 0u);
    // Where the tile's first element lies; the others are at most kDropTile further, which a 32-bit reciprocal divides exactly where a
    // row is shorter than that, and a comparison where it is not.
    int64_t row0 = 0;
    uint32_t col0 = 0;
    if constexpr (!FLAT) {
        row0 = tile0 / g.n_cols;
        col0 = (uint32_t)(tile0 - row0 * g.n_cols);
    }
    const bool full = tile0 + kDropTile <= g.n;  // (uniform)
    auto at = [&](uint32_t i) -> int64_t {
        if constexpr (FLAT) {
            return tile0 + i;
        } else {
            const uint32_t c = col0 + i;
            const uint32_t r = g.n_cols > (uint32_t)kDropTile ? (c >= g.n_cols ? 1u : 0u) : g.n_cols == 1 ? c : __umulhi(c, g.magic);
            return (row0 + r) * g.ldx + (c - r * g.n_cols);
        }
    };
    // fours of elements that neighbour in x too
    const bool whole = FLAT || g.n_cols % 4 == 0;  // (uniform)
    uint32_t quad[kDropQuads];
    float v[kDropQuads][4];
#pragma unroll
    for (int j = 0; j < kDropQuads; ++j) {
        quad[j] = (uint32_t)(j * kBlock + threadIdx.x);
        const uint32_t i = 4 * quad[j];
        if (full && whole) {
            const DropQuad<T> q = *reinterpret_cast<const DropQuad<T>*>(x + at(i));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = DropType<T>::get(q[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = tile0 + i + e < g.n ? DropType<T>::get(x[at(i + e)]) : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < kDropQuads; ++j) {
        const uint64_t ctr = (uint64_t)(tile0 / 4) + quad[j];
        uint32_t words[4] = {0u, 0u, 0u, 0u};
        if (g.threshold != 0) philox4x32_10((uint32_t)ctr, (uint32_t)(ctr >> 32), stream_id, kDropTag, g.seed_lo, g.seed_hi, words);
        const int64_t first = tile0 + 4 * quad[j];
        DropQuad<T> q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = DropType<T>::put(drop_value<RELU>(v[j][e], words[e], g));
        if (full) {
            *reinterpret_cast<DropQuad<T>*>(out + first) = q;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (first + e < g.n) out[first + e] = q[e];
        }
    }
}

// dx = dy / (1 - p) where y, the output of relu and dropout, is not zero (or below: a negative scale there is none)
template <typename T>
__global__ __launch_bounds__(kBlock) void dropout_relu_backward_kernel(const T* __restrict__ dy, const T* __restrict__ y, int64_t n, float scale,
                                                                      T* __restrict__ dx)
{
    const int64_t tile0 = (int64_t)blockIdx.x * kDropTile;
    const bool full = tile0 + kDropTile <= n;
#pragma unroll
    for (int j = 0; j < kDropQuads; ++j) {
        const int64_t i = tile0 + 4 * (int64_t)(j * kBlock + threadIdx.x);
        if (full) {
            const DropQuad<T> a = *reinterpret_cast<const DropQuad<T>*>(dy + i), b = *reinterpret_cast<const DropQuad<T>*>(y + i);
            DropQuad<T> q;
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = DropType<T>::put(DropType<T>::get(b[e]) <= 0.0f ? 0.0f : DropType<T>::get(a[e]) * scale);
            *reinterpret_cast<DropQuad<T>*>(dx + i) = q;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) dx[i + e] = DropType<T>::put(DropType<T>::get(y[i + e]) <= 0.0f ? 0.0f : DropType<T>::get(dy[i + e]) * scale);
        }
    }
}

template <typename T>
void launch_dropout(const DropArgs& g, bool relu, bool flat, unsigned blocks, hipStream_t s)
{
    const dim3 grid(blocks), block(kBlock);
    if (relu && flat) hipLaunchKernelGGL((dropout_kernel<T, true, true>), grid, block, 0, s, g);
    else if (relu) hipLaunchKernelGGL((dropout_kernel<T, true, false>), grid, block, 0, s, g);
    else if (flat) hipLaunchKernelGGL((dropout_kernel<T, false, true>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((dropout_kernel<T, false, false>), grid, block, 0, s, g);
}

}  // namespace fgl

using namespace fgl;

FGL_EXPORT int fgl_dropout(const void* d_x, int64_t ldx, int64_t n_rows, int64_t n_cols, int dtype, double p, uint64_t seed, uint32_t stream_id,
                           const int32_t* d_stream_offset, int relu, void* d_out, void* stream)
{
    FGL_REQUIRE(dtype == FGL_F32 || dtype == FGL_BF16, "dropout: dtype %d", dtype);
    FGL_REQUIRE(p >= 0.0 && p <= 1.0, "dropout: probability %g outside [0, 1]", p);
    FGL_REQUIRE(n_rows >= 0 && n_cols >= 0, "dropout: negative size");
    if (n_rows == 0 || n_cols == 0) return FGL_OK;
    FGL_REQUIRE(d_x && d_out, "dropout: null pointer");
    const bool flat = n_rows == 1 || ldx == n_cols;
    FGL_REQUIRE(flat || ldx > n_cols, "dropout: row stride smaller than the row length");
    FGL_REQUIRE(flat || n_cols < (1LL << 31), "dropout: rows of %lld columns with a stride", (long long)n_cols);
    FGL_REQUIRE(n_rows <= kDropMost / n_cols, "dropout: more than 2^35 elements");
    DropArgs g;
    g.x = d_x;
    g.out = d_out;
    g.n = n_rows * n_cols;
    g.ldx = ldx;
    g.n_cols = flat ? 1 : (uint32_t)n_cols;
    g.magic = flat || n_cols == 1 ? 0u : (uint32_t)(((1ULL << 32) + (uint64_t)n_cols - 1) / (uint64_t)n_cols);
    const double t = nearbyint(p * 4294967296.0);
    g.none = t >= 4294967296.0;
    g.threshold = g.none ? 0xFFFFFFFFu : (uint32_t)t;
    g.stream_id = stream_id;
    g.d_stream_offset = d_stream_offset;
    g.seed_lo = (uint32_t)seed;
    g.seed_hi = (uint32_t)(seed >> 32);
    g.scale = g.none ? 0.0f : (float)(1.0 / (1.0 - p));
    const int64_t blocks = ceil_div(g.n, kDropTile);
    if (dtype == FGL_F32) launch_dropout<float>(g, relu != 0, flat, (unsigned)blocks, as_stream(stream));
    else launch_dropout<__bf16>(g, relu != 0, flat, (unsigned)blocks, as_stream(stream));
    FGL_CHECK_LAUNCH("dropout_kernel");
    return FGL_OK;
}

FGL_EXPORT int fgl_dropout_relu_backward(const void* d_dout, const void* d_out, int64_t n, int dtype, double p, void* d_dx, void* stream)
{
    FGL_REQUIRE(dtype == FGL_F32 || dtype == FGL_BF16, "dropout_relu_backward: dtype %d", dtype);
    FGL_REQUIRE(p >= 0.0 && p <= 1.0, "dropout_relu_backward: probability %g outside [0, 1]", p);
    FGL_REQUIRE(n >= 0 && n <= kDropMost, "dropout_relu_backward: %lld elements", (long long)n);
    if (n == 0) return FGL_OK;
    FGL_REQUIRE(d_dout && d_out && d_dx, "dropout_relu_backward: null pointer");
    const int64_t blocks = ceil_div(n, kDropTile);
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    const dim3 grid((unsigned)blocks), block(kBlock);
    if (dtype == FGL_F32)
        hipLaunchKernelGGL((dropout_relu_backward_kernel<float>), grid, block, 0, as_stream(stream), static_cast<const float*>(d_dout),
                           static_cast<const float*>(d_out), n, scale, static_cast<float*>(d_dx));
    else
        hipLaunchKernelGGL((dropout_relu_backward_kernel<__bf16>), grid, block, 0, as_stream(stream), static_cast<const __bf16*>(d_dout),
                           static_cast<const __bf16*>(d_out), n, scale, static_cast<__bf16*>(d_dx));
    FGL_CHECK_LAUNCH("dropout_relu_backward_kernel");
    return FGL_OK;
}
