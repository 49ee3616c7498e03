// Weight gradient of a dense layer whose input rows are held in 8 bits (fgl_keep8.hpp): C[m, n] = sum over rows r of A[r, m] * step[r, n / 32] code[r, n],
// A the gradient of the layer's output rows; and the column sums of A, the bias gradient.
//
// As fgl_wgrad.hip forms it from rows held in full, with which it shares the split of the rows and the two launches: a wave's 32 VA x 32 VB tile of
// outputs stays in its accumulators, lane i of a half-wave takes VA neighbouring columns of A and VB of the codes of eight rows, which are the operands of
// v_mfma_f32_32x32x16_bf16 as they come, the four waves of a workgroup take every fourth step, their sums are added through LDS and those of the
// workgroups by a second launch in a fixed order.
//
// A code times its step is a bf16 value, so there is nothing to split on that side: fp32 takes three products, of A's three bf16 parts (fgl_split.hpp), instead of six.
// A code becomes one in two and a half instructions: byte to float, one product, two of them rounded to bf16 (exactly) at a time.
// Steps lie by columns, so that a lane has those of its eight rows with one load.
//
// fp32: a step's products are added up from zero before they go to the accumulators, as what a matrix instruction adds is cut to 26 bits of its largest term; every other
// step those of A's negative, since it is cut downwards.  Rows past the end are zeros on both sides.  Where a value of A has bits below 2^-133, bf16's last, that a sum is not
// large beside, or a sum is no number, a workgroup forms its rows again in fp32 instructions.
//
// What bounds it: in fp32 the vector unit (a step of 32 x 128: 44 instructions split A, 104 make the codes' operands, 64 add the products to the accumulators, beside 12 matrix
// instructions of 32 cycles; busy for 55 % and 19 % of the time) and the L2s, from which every tile takes its rows, in bf16 those.  With more than 64 tiles there are
// fewer than eight splits, each of one XCD, and the others have no work: 602 x 512 fp32 runs on six, 1024 x 1024 on two.  us with the second launch: 107 K x 100 x 256 fp32 47 (from rows in full, fgl_wgrad.hip,
// 65; one step ahead instead of two 59, tiles of 64 x 64 52), 8192 x 602 x 256 fp32 30; 87 K x 512 x 256 bf16 52 (tiles of 128 x 64 58).
#include "fgl_column_sums.hpp"
#include "fgl_common.hpp"
#include "fgl_keep8.hpp"
#include "fgl_kernels.hpp"
#include "fgl_split.hpp"
#include "fgl_wgrad8.hpp"

namespace fgl {

typedef float W8F32x16 __attribute__((ext_vector_type(16)));

struct Wgrad8Args {
    const void* a;
    int64_t lda;
    const uint8_t* codes;  // [k][code_ld]
    const uint8_t* steps;  // [code_ld / 32][step_ld]
    int64_t step_ld;
    int code_ld;
    int64_t k;
    int m, n;
    int tiles_n, tiles, splits;
    int64_t k_per_split;
    float* partial;      // [split][tile][register][lane]
    void* c;
    int64_t ldc;
    void* sum_a;         // (may be null)
    float* partial_sum;  // [split][tile along m][column]
};

// Eight rows of V neighbouring columns of A
template <typename T, int V>
struct W8Rows;
template <int V>
struct W8Rows<float, V> {
    typedef float Vec __attribute__((ext_vector_type(V), aligned(4)));
    Vec r[8];
    __device__ __forceinline__ void load(const float* p, int64_t ld)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = *reinterpret_cast<const Vec*>(p + i * ld);
    }
    __device__ __forceinline__ void load_tail(const float* p, int64_t ld, int n)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            r[i] = Vec{};
            if (i < n) r[i] = *reinterpret_cast<const Vec*>(p + i * ld);
        }
    }
    __device__ __forceinline__ void add_columns(float (&sum)[V]) const
    {
#pragma unroll
        for (int c = 0; c < V; ++c) sum[c] += ((r[0][c] + r[1][c]) + (r[2][c] + r[3][c])) + ((r[4][c] + r[5][c]) + (r[6][c] + r[7][c]));
    }
};
template <int V>
struct W8Rows<uint16_t, V> {
    static constexpr int kWords = V == 4 ? 2 : 1;
    typedef uint32_t Vec2 __attribute__((ext_vector_type(2), aligned(4)));
    uint32_t r[8][kWords];
    __device__ __forceinline__ void load_one(const uint16_t* p, int i)
    {
        if constexpr (V == 1) {
            r[i][0] = *p;
        } else if constexpr (V == 2) {
            r[i][0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            const Vec2 v = *reinterpret_cast<const Vec2*>(p);
            r[i][0] = v[0];
            r[i][1] = v[1];
        }
    }
    __device__ __forceinline__ void load(const uint16_t* p, int64_t ld)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_one(p + i * ld, i);
    }
    __device__ __forceinline__ void load_tail(const uint16_t* p, int64_t ld, int n)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int w = 0; w < kWords; ++w) r[i][w] = 0u;
            if (i < n) load_one(p + i * ld, i);
        }
    }
    __device__ __forceinline__ void add_columns(float (&sum)[V]) const
    {
#pragma unroll
        for (int c = 0; c < V; ++c) {
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = __uint_as_float((c & 1) ? r[i][c >> 1] & 0xFFFF0000u : r[i][c >> 1] << 16);
            sum[c] += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
        }
    }
};

// Eight rows of V neighbouring columns of codes, and the steps of the rows there
template <int V>
struct W8Codes {
    uint32_t r[8];
    uint32_t steps[2];
    __device__ __forceinline__ void load_one(const uint8_t* p, int i)
    {
        if constexpr (V == 1) r[i] = *p;
        else if constexpr (V == 2) r[i] = *reinterpret_cast<const uint16_t*>(p);
        else r[i] = *reinterpret_cast<const uint32_t*>(p);
    }
    __device__ __forceinline__ void load_steps(const uint8_t* s)
    {
        const uint2 v = *reinterpret_cast<const uint2*>(s);
        steps[0] = v.x;
        steps[1] = v.y;
    }
    __device__ __forceinline__ void load(const uint8_t* p, int ld, const uint8_t* s)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_one(p + (int64_t)i * ld, i);
        load_steps(s);
    }
    // only the first n rows exist; a step of zero makes zeros of the others
    __device__ __forceinline__ void load_tail(const uint8_t* p, int ld, const uint8_t* s, int n)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            r[i] = 0;
            if (i < n) load_one(p + (int64_t)i * ld, i);
        }
        load_steps_tail(s, n);
    }
    __device__ __forceinline__ void load_steps_tail(const uint8_t* s, int n)
    {
        steps[0] = steps[1] = 0;
        if (n > 0) load_steps(s);
        if (n < 4) steps[0] &= n <= 0 ? 0u : (1u << 8 * n) - 1u;
        if (n < 8) steps[1] &= n <= 4 ? 0u : (1u << 8 * (n - 4)) - 1u;
    }
    __device__ __forceinline__ float value(int i, int c) const { return k8_code_value(r[i], c) * k8_step_value(steps[i / 4] >> 8 * (i % 4) & 0xFFu); }
    // column c of the eight rows, as the matrix instruction's operand
    __device__ __forceinline__ void columns(SpU4 (&to)[V]) const
    {
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = k8_step_value(steps[i / 4] >> 8 * (i % 4) & 0xFFu);
#pragma unroll
        for (int c = 0; c < V; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                typedef __bf16 B2 __attribute__((ext_vector_type(2)));
                B2 h;
                h[0] = (__bf16)(k8_code_value(r[2 * j], c) * s[2 * j]);
                h[1] = (__bf16)(k8_code_value(r[2 * j + 1], c) * s[2 * j + 1]);
                to[c][j] = __builtin_bit_cast(uint32_t, h);
            }
    }
};

// first column of lane i's vector (i in 0..31) in a tile of A; a lane whose columns would leave the row takes the last ones again
template <int V>
__device__ __forceinline__ int w8_column(int tile, int i, int m)
{
    const int c = (tile * 32 + i) * V;
    return c + V <= m ? c : m - V;
}

// Where a wave's lanes read: rows first, first + kStep, ..; col_a, col_b: the lane's first columns
template <typename T, int VB>
struct W8Walk {
    static constexpr int64_t kStep = 16 * (kBlock / kWave);
    const T* a;
    const uint8_t* codes;
    const uint8_t* steps;
    int at = 0;
    int whole, last_rows;  // steps before the last one, which has so many rows of the lane's eight (none or fewer than none, it may be)
    __device__ __forceinline__ W8Walk(const Wgrad8Args& g, int64_t k0, int64_t k1, int wave, int col_a, int col_b)
    {
        const int half = lane_id() / 32;
        const int64_t first = k0 + 16 * wave;
        whole = k1 > first ? (int)((k1 - first - 1) / kStep) : 0;
        const int64_t left = k1 - (first + whole * kStep) - 8 * half;
        last_rows = left > 8 ? 8 : left < 0 ? 0 : (int)left;
        const int64_t row = first + 8 * half;
        a = static_cast<const T*>(g.a) + row * g.lda + col_a;
        codes = g.codes + row * g.code_ld + col_b;
        steps = g.steps + (int64_t)(col_b / 32) * g.step_ld + row;
    }
    // the steps in order: the whole ones (at least one; after the last, that one again), the last one
    template <int VA>
    __device__ __forceinline__ void load(const Wgrad8Args& g, W8Rows<T, VA>& ra, W8Codes<VB>& rb)
    {
        ra.load(a, g.lda);
        rb.load(codes, g.code_ld, steps);
        advance(g, ++at < whole ? kStep : 0);
    }
    template <int VA>
    __device__ __forceinline__ void load_tail(const Wgrad8Args& g, W8Rows<T, VA>& ra, W8Codes<VB>& rb)
    {
        if (whole > 0) advance(g, kStep);
        ra.load_tail(a, g.lda, last_rows);
        rb.load_tail(codes, g.code_ld, steps, last_rows);
    }
    __device__ __forceinline__ void load_steps(int i, W8Codes<VB>& rb)
    {
        rb.load_steps_tail(steps, i < whole ? 8 : last_rows);
        steps += kStep;
    }
    __device__ __forceinline__ void advance(const Wgrad8Args& g, int64_t rows)
    {
        a += rows * g.lda;
        codes += rows * g.code_ld;
        steps += rows;
    }
};

// acc += the products of the wave's rows, in fp32 instructions
template <int VA, int VB>
__device__ __forceinline__ void w8_plain(const Wgrad8Args& g, int64_t k0, int64_t k1, int wave, int col_a, int col_b, W8F32x16 (&acc)[VA * VB])
{
    W8Walk<float, VB> walk(g, k0, k1, wave, col_a, col_b);
    W8Rows<float, VA> a;
    W8Codes<VB> b;
    for (int i = 0; i <= walk.whole; ++i) {
        if (i < walk.whole) walk.load(g, a, b);
        else walk.load_tail(g, a, b);
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int p = 0; p < VA; ++p)
#pragma unroll
                for (int q = 0; q < VB; ++q) acc[p * VB + q] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.r[r][p], b.value(r, q), acc[p * VB + q], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < VA * VB; ++t) {
        // (no branch between the last products and the first reads)
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(0.0f, 0.0f, acc[t], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = acc[t][i] + 0.0f;
            asm volatile("" : "+v"(s));
            acc[t][i] = s;
        }
    }
}

// The wave's rows in parts; true where the lane met values that have none (then acc is not the sum)
template <int VA, int VB>
__device__ __forceinline__ bool w8_rows(const Wgrad8Args& g, int64_t k0, int64_t k1, int wave, int col_a, int col_b, bool sums, W8F32x16 (&acc)[VA * VB], float (&sum)[VA])
{
    constexpr int kAhead = 2;
    const int half = lane_id() / 32;
    W8Walk<float, VB> walk(g, k0, k1, wave, col_a, col_b);
    W8Rows<float, VA> a[kAhead];
    W8Codes<VB> b[kAhead];
    uint32_t rest[VA];
#pragma unroll
    for (int i = 0; i < VA; ++i) rest[i] = 0;
    float sign = 1.0f;
    auto multiply = [&](const W8Rows<float, VA>& ra, const W8Codes<VB>& rb, auto&& then) {
        if (sums) ra.add_columns(sum);
        SpU4 pa[VA][3], pb[VB];
        rb.columns(pb);
#pragma unroll
        for (int i = 0; i < VA; ++i) {
            float v[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = ra.r[r][i] * sign;
            sp_split<true>(v, pa[i], rest[i]);
        }
        then();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < VA; ++i) {
            W8F32x16 part[VB];
#pragma unroll
            for (int q = 2; q >= 0; --q)  // (the small products first)
#pragma unroll
                for (int j = 0; j < VB; ++j)
                    part[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf16x8, pa[i][q]), __builtin_bit_cast(Bf16x8, pb[j]), q == 2 ? W8F32x16{} : part[j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < VB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i * VB + j][r] = fmaf(part[j][r], sign, acc[i * VB + j][r]);
        }
        sign = -sign;
    };
    // (nothing branches around the loads: past the last whole step that one is read again, and not used)
    if (walk.whole > 0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) walk.load(g, a[u], b[u]);
        int s = 0;
        for (; s + kAhead <= walk.whole; s += kAhead)
#pragma unroll
            for (int u = 0; u < kAhead; ++u) multiply(a[u], b[u], [&] { walk.load(g, a[u], b[u]); });
#pragma unroll
        for (int u = 0; u + 1 < kAhead; ++u)
            if (s + u < walk.whole) multiply(a[u], b[u], [] {});
    }
    walk.load_tail(g, a[0], b[0]);
    multiply(a[0], b[0], [] {});
    bool odd = false;
#pragma unroll
    for (int t = 0; t < VA * VB; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) odd |= sp_odd(acc[t][i]);
    bool loses = false;
#pragma unroll
    for (int i = 0; i < VA; ++i) {
        rest[i] = (rest[i] | __shfl_xor(rest[i], 32, kWave)) & 0xFFFFu;
        loses |= rest[i] != 0;
    }
    if (__any(loses)) {
        // the largest value that the lane's codes may stand for, from their steps
        W8Walk<float, VB> again(g, k0, k1, wave, col_a, col_b);
        uint32_t most = 0;
        for (int s = 0; s <= again.whole; ++s) {
            W8Codes<VB> t;
            again.load_steps(s, t);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const uint32_t v = t.steps[r / 4] >> 8 * (r % 4) & 0xFFu;
                most = most > v ? most : v;
            }
        }
        const float value = __uint_as_float(most << 23) * 128.0f;
        const float largest = fmaxf(value, __shfl_xor(value, 32, kWave)), terms = (float)(walk.whole + 1) * 16.0f;
#pragma unroll
        for (int i = 0; i < VA; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool row_loses = __shfl((int)rest[i], 8 * (r / 4) + 4 * half + r % 4, kWave) != 0;  // (of the lane with that column of A)
#pragma unroll
                for (int j = 0; j < VB; ++j) odd |= !(fabsf(acc[i * VB + j][r]) >= sp_least(terms, row_loses, 0.0f, false, largest));
            }
    }
    return odd;
}

// The wave's rows in bf16.  Steps are on their way three ahead of the one that is multiplied.  (87 K x 512 x 256: in tiles of 128 x 128, one wave a SIMD and one step ahead, 65 us,
// 128 x 64 so 53, 64 x 128 47.)
template <int VA, int VB, bool SUMS>
__device__ __forceinline__ void w8_rows(const Wgrad8Args& g, int64_t k0, int64_t k1, int wave, int col_a, int col_b, W8F32x16 (&acc)[VA * VB], float (&sum)[VA])
{
    constexpr int kAhead = 3;
    W8Walk<uint16_t, VB> walk(g, k0, k1, wave, col_a, col_b);
    W8Rows<uint16_t, VA> a[kAhead];
    W8Codes<VB> b[kAhead];
    auto multiply = [&](const W8Rows<uint16_t, VA>& ra, const W8Codes<VB>& rb, auto&& then) {
        if constexpr (SUMS) ra.add_columns(sum);
        SpU4 pa[VA], pb[VB];
        rb.columns(pb);
#pragma unroll
        for (int i = 0; i < VA; ++i) pa[i] = __builtin_bit_cast(SpU4, bf16_column(ra.r, i));
        then();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < VA; ++i)
#pragma unroll
            for (int j = 0; j < VB; ++j)
                acc[i * VB + j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf16x8, pa[i]), __builtin_bit_cast(Bf16x8, pb[j]), acc[i * VB + j], 0, 0, 0);
    };
    // (nothing branches around the loads: past the last whole step that one is read again, and not used)
    if (walk.whole > 0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) walk.load(g, a[u], b[u]);
        int s = 0;
        for (; s + kAhead <= walk.whole; s += kAhead)
#pragma unroll
            for (int u = 0; u < kAhead; ++u) multiply(a[u], b[u], [&] { walk.load(g, a[u], b[u]); });
#pragma unroll
        for (int u = 0; u + 1 < kAhead; ++u)
            if (s + u < walk.whole) multiply(a[u], b[u], [] {});
    }
    walk.load_tail(g, a[0], b[0]);
    multiply(a[0], b[0], [] {});
#pragma unroll
    for (int t = 0; t < VA * VB; ++t)  // (no branch between the last products and the first reads)
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Bf16x8{}, Bf16x8{}, acc[t], 0, 0, 0);
#pragma unroll
    for (int t = 0; t < VA * VB; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v = acc[t][i] + 0.0f;
            asm volatile("" : "+v"(v));
            acc[t][i] = v;
        }
}

template <typename T, int VA, int VB>
__global__ __launch_bounds__(kBlock, 2) void wgrad8_kernel(const Wgrad8Args g)
{
    constexpr int kTiles = VA * VB, kChunk = kTiles < 4 ? kTiles : 4, kWaves = kBlock / kWave;
    __shared__ float s_acc[kWaves][kChunk * 16][kWave];
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));  // (branches around matrix instructions are the whole wave's)
    // workgroup -> (split, tile): eight neighbouring splits (one per XCD) take turns, so the tiles of a split share an XCD
    const int group = (int)(blockIdx.x / (8u * (unsigned)g.tiles)), in_group = (int)(blockIdx.x % (8u * (unsigned)g.tiles));
    const int split = group * 8 + in_group % 8, tile = in_group / 8;
    if (split >= g.splits) return;  // (uniform over the workgroup)
    const int tm = tile / g.tiles_n, tn = tile % g.tiles_n;
    const int64_t k0 = (int64_t)split * g.k_per_split;
    const int64_t k1 = k0 + g.k_per_split < g.k ? k0 + g.k_per_split : g.k;
    const int col_a = w8_column<VA>(tm, lane % 32, g.m);
    const int own_b = (tn * 32 + lane % 32) * VB, col_b = own_b + VB <= g.code_ld ? own_b : g.code_ld - VB;
    W8F32x16 acc[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) acc[t] = W8F32x16{};
    const bool sums = g.sum_a != nullptr && tn == 0;
    float sum[VA];
#pragma unroll
    for (int i = 0; i < VA; ++i) sum[i] = 0.0f;
    if constexpr (sizeof(T) == 4) {
        if (__syncthreads_or(w8_rows<VA, VB>(g, k0, k1, wave, col_a, col_b, sums, acc, sum))) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t) acc[t] = W8F32x16{};
            w8_plain<VA, VB>(g, k0, k1, wave, col_a, col_b, acc);
        }
    } else {
        if (sums) w8_rows<VA, VB, true>(g, k0, k1, wave, col_a, col_b, acc, sum);
        else w8_rows<VA, VB, false>(g, k0, k1, wave, col_a, col_b, acc, sum);
    }
    float* out = g.partial + ((int64_t)split * g.tiles + tile) * (kTiles * 16) * kWave;
#pragma unroll
    for (int q = 0; q < kTiles / kChunk; ++q) {
#pragma unroll
        for (int t = 0; t < kChunk; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s_acc[wave][t * 16 + i][lane] = acc[q * kChunk + t][i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kChunk * 4; ++i) {  // each wave adds up a quarter of the registers
            const int r = wave * (kChunk * 4) + i;
            float s = s_acc[0][r][lane];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) s += s_acc[w][r][lane];
            out[(int64_t)(q * kChunk * 16 + r) * kWave + lane] = s;
        }
        __syncthreads();
    }
    if (!sums) return;
    float* s_sum = &s_acc[0][0][0];
#pragma unroll
    for (int i = 0; i < VA; ++i) {
        const float s = sum[i] + __shfl_xor(sum[i], 32, kWave);  // (the half-waves hold different rows of the same columns)
        if (lane < 32) s_sum[wave * (32 * VA) + lane * VA + i] = s;
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < 32 * VA; i += kBlock) {
        float s = s_sum[i];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) s += s_sum[w * (32 * VA) + i];
        g.partial_sum[((int64_t)split * (g.tiles / g.tiles_n) + tm) * (32 * VA) + i] = s;
    }
}

// Adds the splits: a workgroup per (tile, accumulator register), four lanes of splits per output; behind those, a workgroup per 64 column sums of A.
template <typename T, int VA, int VB>
__global__ __launch_bounds__(kBlock) void wgrad8_reduce_kernel(const Wgrad8Args g)
{
    constexpr int kTiles = VA * VB, kWaves = kBlock / kWave;
    __shared__ float s_sum[kWaves][kWave];
    const int lane = lane_id(), wave = (int)(threadIdx.x / kWave);
    const int tile = (int)(blockIdx.x / (kTiles * 16)), reg = (int)(blockIdx.x % (kTiles * 16));
    const bool sums = tile >= g.tiles;  // (uniform over the workgroup)
    const int sum_columns = g.tiles / g.tiles_n * 32 * VA;
    const int at = (int)(blockIdx.x - (unsigned)(g.tiles * kTiles * 16)) * kWave + lane;  // column sums only
    const int64_t stride = sums ? sum_columns : (int64_t)g.tiles * (kTiles * 16) * kWave;
    const float* p = sums ? g.partial_sum + (at < sum_columns ? at : 0) : g.partial + ((int64_t)tile * (kTiles * 16) + reg) * kWave + lane;
    float s = 0.0f;
    int q = wave;
    for (; q + 3 * kWaves < g.splits; q += 4 * kWaves) {
        const float v0 = p[q * stride], v1 = p[(q + kWaves) * stride], v2 = p[(q + 2 * kWaves) * stride], v3 = p[(q + 3 * kWaves) * stride];
        s += (v0 + v1) + (v2 + v3);
    }
    for (; q < g.splits; q += kWaves) s += p[q * stride];
    s_sum[wave][lane] = s;
    __syncthreads();
    if (wave != 0) return;
    s = (s_sum[0][lane] + s_sum[1][lane]) + (s_sum[2][lane] + s_sum[3][lane]);
    if (sums) {
        if (at >= sum_columns) return;
        const int col = w8_column<VA>(at / (32 * VA), at % (32 * VA) / VA, g.m) + at % VA;
        if constexpr (sizeof(T) == 4) static_cast<float*>(g.sum_a)[col] = s;
        else static_cast<__bf16*>(g.sum_a)[col] = (__bf16)s;
        return;
    }
    // accumulator register r of lane l: row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32 of its 32x32 tile
    const int r = reg % 16, t = reg / 16;
    const int row = 8 * (r / 4) + 4 * (lane / 32) + r % 4;
    const int own_m = (tile / g.tiles_n * 32 + row) * VA, mm = w8_column<VA>(tile / g.tiles_n, row, g.m) + t / VB;
    const int nn = (tile % g.tiles_n * 32 + lane % 32) * VB + t % VB;
    if (nn >= g.n) return;  // (columns of the codes that fill up a step's 32, and repeated ones)
    if (mm < own_m) return;  // (repeated columns of A: one may be another tile's, whose sum has other bits where only one of the two formed its rows again)
    if constexpr (sizeof(T) == 4) static_cast<float*>(g.c)[(int64_t)mm * g.ldc + nn] = s;
    else static_cast<__bf16*>(g.c)[(int64_t)mm * g.ldc + nn] = (__bf16)s;
}

// Columns a lane along one side: what pads the least, the wider of two that pad alike (a fifth more is a fair price for a load twice as wide)
static int w8_vec(int n, bool vectors, int widest)
{
    if (!vectors || n <= 32) return 1;
    int best = 1;
    int64_t pad = ceil_div(n, 32) * 32;
    for (int v = 2; v <= widest; v *= 2) {
        const int64_t p = ceil_div(n, 32 * v) * 32 * v;
        if (n >= v && p * 10 <= pad * 12) {
            best = v;
            if (p < pad) pad = p;
        }
    }
    return best;
}

struct Wgrad8Plan {
    int va, vb, tiles_n, tiles, splits;
    int64_t k_per_split;
    size_t sum_offset, ws_bytes;
};

static Wgrad8Plan w8_plan(int64_t k, int m, int n, int dtype, bool vectors)
{
    Wgrad8Plan p;
    // codes are the fewer bytes: a tile is wide in them, and narrow in A where both could be
    p.vb = w8_vec((int)k8_columns(n), true, 4);
    p.va = w8_vec(m, vectors, dtype == FGL_F32 ? (p.vb == 4 ? 1 : 2) : (p.vb == 4 ? 2 : 4));
    p.tiles_n = (int)ceil_div(n, 32 * p.vb);
    p.tiles = p.tiles_n * (int)ceil_div(m, 32 * p.va);
    const int per_cu = dtype == FGL_F32 || p.va * p.vb >= 8 ? 2 : 4;
    int64_t splits = 256 * per_cu / p.tiles;
    const int64_t most = ceil_div(k, 256);  // 256 rows and more a split: the sum over the splits costs as much as they do otherwise
    if (splits > most) splits = most;
    if (splits > 8) splits = splits / 8 * 8;
    if (splits < 1) splits = 1;
    p.k_per_split = ceil_div(ceil_div(k, splits), 64) * 64;
    if (p.k_per_split < 64) p.k_per_split = 64;
    p.splits = (int)ceil_div(k, p.k_per_split);
    if (p.splits < 1) p.splits = 1;
    p.sum_offset = align_up((size_t)p.splits * p.tiles * p.va * p.vb * 16 * kWave * sizeof(float), 256);
    p.ws_bytes = p.sum_offset + align_up((size_t)p.splits * (p.tiles / p.tiles_n) * 32 * p.va * sizeof(float), 256);
    return p;
}

size_t wgrad8_workspace_bytes(int64_t k, int m, int n, int dtype)
{
    const size_t a = w8_plan(k, m, n, dtype, true).ws_bytes, b = w8_plan(k, m, n, dtype, false).ws_bytes;
    return a > b ? a : b;
}

ColumnSplit wgrad8_column_split(int64_t k, int m, int n, int dtype)
{
    const Wgrad8Plan p = w8_plan(k, m, n, dtype, dtype == FGL_F32 || m % 2 == 0);
    return {p.splits, p.k_per_split, false};
}

template <typename T, int VA, int VB>
static void launch_wgrad8(const Wgrad8Args& g, hipStream_t stream)
{
    const int64_t blocks = ceil_div(g.splits, 8) * 8 * g.tiles;
    hipLaunchKernelGGL((wgrad8_kernel<T, VA, VB>), dim3((unsigned)blocks), dim3(kBlock), 0, stream, g);
    const int64_t sum_blocks = g.sum_a != nullptr ? ceil_div((int64_t)(g.tiles / g.tiles_n) * 32 * VA, kWave) : 0;
    hipLaunchKernelGGL((wgrad8_reduce_kernel<T, VA, VB>), dim3((unsigned)(g.tiles * VA * VB * 16 + sum_blocks)), dim3(kBlock), 0, stream, g);
}

int launch_wgrad8(const void* a, int64_t lda, const uint8_t* codes, const uint8_t* steps, int64_t k, int m, int n, int dtype, void* c, int64_t ldc, void* sum_a, void* ws,
                  size_t ws_bytes, hipStream_t stream)
{
    const Wgrad8Plan p = w8_plan(k, m, n, dtype, dtype == FGL_F32 || (m % 2 == 0 && lda % 2 == 0 && ((uintptr_t)a & 3) == 0));
    if (ws == nullptr || ws_bytes < p.ws_bytes) {
        set_error("weight gradient: workspace too small (%zu < %zu)", ws_bytes, p.ws_bytes);
        return FGL_ERR_WORKSPACE;
    }
    Wgrad8Args g;
    memset(&g, 0, sizeof(g));
    g.a = a; g.lda = lda; g.codes = codes; g.steps = steps; g.step_ld = w8_step_ld(k); g.code_ld = (int)k8_columns(n); g.k = k; g.m = m; g.n = n;
    g.tiles_n = p.tiles_n; g.tiles = p.tiles; g.splits = p.splits; g.k_per_split = p.k_per_split; g.partial = static_cast<float*>(ws); g.c = c; g.ldc = ldc;
    g.sum_a = sum_a; g.partial_sum = reinterpret_cast<float*>(static_cast<char*>(ws) + p.sum_offset);
    auto wide = [&](auto type) {
        using T = decltype(type);
        if constexpr (sizeof(T) == 2) {
            if (p.va == 4 && p.vb == 2) return launch_wgrad8<T, 4, 2>(g, stream);
            if (p.va == 4) return launch_wgrad8<T, 4, 1>(g, stream);
            if (p.va == 2 && p.vb == 4) return launch_wgrad8<T, 2, 4>(g, stream);
        }
        if (p.vb == 4) return launch_wgrad8<T, 1, 4>(g, stream);
        if (p.va == 2 && p.vb == 2) return launch_wgrad8<T, 2, 2>(g, stream);
        if (p.va == 2) return launch_wgrad8<T, 2, 1>(g, stream);
        if (p.vb == 2) return launch_wgrad8<T, 1, 2>(g, stream);
        return launch_wgrad8<T, 1, 1>(g, stream);
    };
    if (dtype == FGL_F32) wide(float{});
    else wide(uint16_t{});
    FGL_CHECK_LAUNCH("wgrad8_kernel");
    return FGL_OK;
}

}  // namespace fgl
