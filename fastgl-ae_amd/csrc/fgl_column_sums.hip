// Sums over the rows of A[k, m], column by column: the gradient of a layer's bias where its weight has none.  (Beside the weight's it costs fgl_wgrad.hip's and
// fgl_wgrad8.hip's kernels nothing, which have the rows in registers.)
//
// A column's terms are added in the order in which those kernels add them, so that a bias's gradient has the same bits whether or not its weight has one: the rows
// are split as theirs are, the four waves of a workgroup take every fourth step of a split, a half-wave half of a step's rows, then halves, waves and splits are
// added, the splits by a second launch.  Only the columns of a lane are this file's to choose: two neighbours where they are one load.
//
// What bounds it: the pass over A, with four steps (32 rows a lane) on their way, by as many workgroups as that order leaves: 60 K x 256 fp32 13 us (4.6 TB/s), 87 K x 512 bf16 18 (5.0),
// 2.4 M x 64 bf16 75 (4.1), and 3 to 12 for the second launch; 100 K x 1024 bf16 beside 1024 columns of x, in four splits, 99 (2.1).
#include "fgl_column_sums.hpp"
#include "fgl_common.hpp"

#include <type_traits>

namespace fgl {

constexpr int kCsAhead = 4;  // steps on their way together

struct ColumnSumsArgs {
    const void* a;
    int64_t lda, k;
    int m, tiles, splits;  // tiles of 32 V columns
    int64_t k_per_split;
    float* partial;  // [split][column]
    void* out;
};

template <typename T, int V>
struct CsLoad;
template <int V>
struct CsLoad<float, V> {
    typedef float Vec __attribute__((ext_vector_type(V), aligned(4)));
    Vec v;
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const Vec*>(p); }
    __device__ __forceinline__ void zero() { v = Vec{}; }
    __device__ __forceinline__ float at(int c) const { return v[c]; }
};
template <int V>
struct CsLoad<uint16_t, V> {
    uint32_t v;
    __device__ __forceinline__ void load(const uint16_t* p)
    {
        if constexpr (V == 2) v = *reinterpret_cast<const uint32_t*>(p);
        else v = *p;
    }
    __device__ __forceinline__ void zero() { v = 0; }
    __device__ __forceinline__ float at(int c) const { return __uint_as_float(c ? v & 0xFFFF0000u : v << 16); }
};

// V == 2: rows of two columns and more, in bf16 whole words (every row starts on one)
template <typename T, int V, bool EVERY_OTHER>
__global__ __launch_bounds__(kBlock) void column_sums_kernel(const ColumnSumsArgs g)
{
    constexpr int kWaves = kBlock / kWave, N = EVERY_OTHER ? 4 : 8;  // rows of a lane in a step
    constexpr int64_t kStep = 2 * N * kWaves;
    __shared__ float s_sum[kWaves][32 * V];
    const int lane = lane_id(), half = lane / 32, wave = (int)(threadIdx.x / kWave);
    const int split = (int)blockIdx.x / g.tiles, tile = (int)blockIdx.x % g.tiles;
    const int64_t k0 = (int64_t)split * g.k_per_split, k1 = k0 + g.k_per_split < g.k ? k0 + g.k_per_split : g.k;
    const int own = (tile * 32 + lane % 32) * V, col = own + V <= g.m ? own : g.m - V;
    const int64_t first = k0 + 2 * N * wave;
    const int whole = k1 > first ? (int)((k1 - first - 1) / kStep) : 0;  // steps before the last one, which may be short or empty
    const T* p = static_cast<const T*>(g.a) + (first + (EVERY_OTHER ? half : N * half)) * g.lda + col;
    auto row = [&](int s, int i) { return p + (s * kStep + (EVERY_OTHER ? 2 * i : i)) * g.lda; };
    float sum[V];
#pragma unroll
    for (int c = 0; c < V; ++c) sum[c] = 0.0f;
    auto add = [&](const CsLoad<T, V> (&r)[N]) {
#pragma unroll
        for (int c = 0; c < V; ++c) {
            float s = (r[0].at(c) + r[1].at(c)) + (r[2].at(c) + r[3].at(c));
            if constexpr (N == 8) s += (r[4].at(c) + r[5].at(c)) + (r[6].at(c) + r[7].at(c));
            sum[c] += s;
        }
    };
    int s = 0;
    for (; s + kCsAhead <= whole; s += kCsAhead) {
        CsLoad<T, V> r[kCsAhead][N];
#pragma unroll
        for (int u = 0; u < kCsAhead; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) r[u][i].load(row(s + u, i));
#pragma unroll
        for (int u = 0; u < kCsAhead; ++u) add(r[u]);
    }
    for (; s < whole; ++s) {
        CsLoad<T, V> r[N];
#pragma unroll
        for (int i = 0; i < N; ++i) r[i].load(row(s, i));
        add(r);
    }
    const int64_t last = first + whole * kStep;
    CsLoad<T, V> r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        r[i].zero();
        if (last + (EVERY_OTHER ? 2 * i + half : N * half + i) < k1) r[i].load(row(whole, i));
    }
    add(r);
#pragma unroll
    for (int c = 0; c < V; ++c) {
        const float both = sum[c] + __shfl_xor(sum[c], 32, kWave);
        if (lane < 32) s_sum[wave][lane * V + c] = both;
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < 32 * V; i += kBlock) {
        float t = s_sum[0][i];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) t += s_sum[w][i];
        g.partial[((int64_t)split * g.tiles + tile) * (32 * V) + i] = t;
    }
}

// Adds the splits: 64 columns a workgroup, a wave every fourth split
template <typename T, int V>
__global__ __launch_bounds__(kBlock) void column_sums_reduce_kernel(const ColumnSumsArgs g)
{
    constexpr int kWaves = kBlock / kWave;
    __shared__ float s_sum[kWaves][kWave];
    const int lane = lane_id(), wave = (int)(threadIdx.x / kWave), columns = g.tiles * 32 * V, at = (int)blockIdx.x * kWave + lane;
    const float* p = g.partial + (at < columns ? at : 0);
    const int64_t stride = columns;
    float s = 0.0f;
    int q = wave;
    for (; q + 3 * kWaves < g.splits; q += 4 * kWaves) {
        const float v0 = p[q * stride], v1 = p[(q + kWaves) * stride], v2 = p[(q + 2 * kWaves) * stride], v3 = p[(q + 3 * kWaves) * stride];
        s += (v0 + v1) + (v2 + v3);
    }
    for (; q < g.splits; q += kWaves) s += p[q * stride];
    s_sum[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || at >= columns) return;
    s = (s_sum[0][lane] + s_sum[1][lane]) + (s_sum[2][lane] + s_sum[3][lane]);
    const int own = at / V * V, col = (own + V <= g.m ? own : g.m - V) + at % V;
    if (col < own) return;  // (repeated: its neighbour's)
    if constexpr (sizeof(T) == 4) static_cast<float*>(g.out)[col] = s;
    else static_cast<__bf16*>(g.out)[col] = (__bf16)s;
}

static int cs_tiles(int m, int v) { return (int)ceil_div(m, 32 * v); }

size_t column_sums_workspace_bytes(const ColumnSplit& split, int m) { return align_up((size_t)split.splits * cs_tiles(m, 2) * 64 * sizeof(float), 256); }

int launch_column_sums(const void* a, int64_t lda, int64_t k, int m, int dtype, const ColumnSplit& split, void* out, void* ws, size_t ws_bytes, hipStream_t stream)
{
    if (ws == nullptr || ws_bytes < column_sums_workspace_bytes(split, m)) {
        set_error("column sums: workspace too small (%zu < %zu)", ws_bytes, column_sums_workspace_bytes(split, m));
        return FGL_ERR_WORKSPACE;
    }
    const bool two = dtype == FGL_F32 ? m >= 2 : m % 2 == 0;
    ColumnSumsArgs g{a, lda, k, m, cs_tiles(m, two ? 2 : 1), split.splits, split.k_per_split, static_cast<float*>(ws), out};
    auto launch = [&](auto type, auto wide, auto every_other) {
        using T = decltype(type);
        constexpr int V = decltype(wide)::value;
        hipLaunchKernelGGL((column_sums_kernel<T, V, decltype(every_other)::value>), dim3((unsigned)(g.splits * g.tiles)), dim3(kBlock), 0, stream, g);
        hipLaunchKernelGGL((column_sums_reduce_kernel<T, V>), dim3((unsigned)ceil_div(g.tiles * 32 * V, kWave)), dim3(kBlock), 0, stream, g);
    };
    auto of = [&](auto type, auto every_other) {
        if (two) launch(type, std::integral_constant<int, 2>{}, every_other);
        else launch(type, std::integral_constant<int, 1>{}, every_other);
    };
    if (dtype == FGL_BF16) of(uint16_t{}, std::false_type{});
    else if (split.every_other) of(float{}, std::true_type{});
    else of(float{}, std::false_type{});
    FGL_CHECK_LAUNCH("column_sums_kernel");
    return FGL_OK;
}

}  // namespace fgl
