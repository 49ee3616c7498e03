// Softmax cross entropy of a dense layer's rows, with its gradients, without the logits ever lying in memory: for rows x_i (D
// columns), classes w_v with biases b_v and labels y_i
//   s_iv = x_i . w_v + b_v,   loss_i = log sum_v exp(s_iv) - s_iy,   p_iv = exp(s_iv) / sum_v exp(s_iv)
//   dx_i = g_i (sum_{v != y} p_iv w_v - (1 - p_iy) w_y)
//   dw_v = sum_{i: y_i != v} g_i p_iv x_i - sum_{i: y_i = v} g_i (1 - p_iy) x_i,   db_v the same with 1 in the place of x_i.
// g_i is the gradient of loss_i.  1 - p_iy is formed as the other classes' share of the sum, and the loss as log(1 + others / own), so
// that rows that are certain of their label keep all their bits.
//
// One kernel, three uses (xe_kernel).  A wave keeps 32 rows of one matrix ("kept") and passes over tiles of 32 rows of the other
// ("passed"): S^T = passed kept^T by matrix instructions, P^T = exp of it, and O^T += passed^T P^T.
//   loss alone:   kept = x, passed = w, no O          loss and dx:   kept = x, passed = w, O = sum of p w          dw:   kept = w, passed = x
// dx is formed in the forward pass, where p is at hand (up to its factor g_i), so the logits are formed twice in all: 8 N V D operations.
// S^T rather than S: a lane of a matrix result has one column, so a lane has one kept row -- its running maximum, sum and
// rescaling are the lane's own -- and the sixteen values of S^T that it has are, rounded, an operand of the second product as they
// are (its k, the passed rows, is taken in the order in which the lanes have it).  O^T for the same reason.
// The running maximum is moved only where a row's largest value passes it by 2^8 (fp32 and bf16 hold p up to there with
// the same relative error), so that O is rescaled a few times a pass and not once a tile.
//
// Operands: "images" (xe_images_kernel), a copy of x and w in the order in which the lanes take them, 1 KB for each 32 x 16 values, rows
// and columns padded with zeros: once as operand of S (lane: row, eight columns) and once of O (lane: column, eight rows).  So a tile is
// copied to LDS straight, without a register or a bank conflict, and no access is out of bounds whatever the sizes.  A tile's
// first kilobyte has what belongs to its 32 rows: biases, or labels and the backward pass's factors.
//
// fp32: each value in three bf16 parts (fgl_split.hpp), six matrix instructions a product, their sum over 32 k added to fp32 accumulators.
// bf16: P and the results are rounded to bf16, as the operands are; sums, maxima and losses are fp32 in both.
// Values must be finite, and below 3.38e38 in fp32, where a part would round to infinity: others make losses and gradients that are not
// numbers.  A bias of -1e30 or less, -infinity among them, leaves its class out: no share, no gradient.  (Shares are exp2 of one fma, whose
// product with log2 e is not rounded where the maximum's is: logits up to some 1e9 are no matter, the difference of 2^-25 of the maximum is the
// same for all of a row's shares and their sum.)
//
// Split: the passed rows are shared among `splits` workgroups so that the chip is full; each leaves its O, maximum and sum in
// scratch, and xe_combine adds them up in order (the same bits on every run).
#include "fgl_common.hpp"
#include "fgl_kernels.hpp"
#include "fgl_split.hpp"

#include <math.h>

namespace fgl {

typedef float XeF4 __attribute__((ext_vector_type(4)));

constexpr int kXeWaves = kBlock / kWave;
constexpr int kXeChunk = 1024;  // bytes of an operand of one matrix instruction
constexpr int kXeMaxSplits = 64;
constexpr int kXeMaxDim = 512;
constexpr float kXeLog2e = 1.44269504088896340736f;
constexpr float kXeLn2 = 0.69314718055994530942f;
constexpr float kXeLeftOut = -1e30f;  // a bias of this or less leaves its class out, as -infinity does
constexpr float kXeStep = 8.0f;       // powers of two that a row's values may pass its running maximum by

enum { kXeLoss = 0, kXeLossAndRows = 1, kXeWeights = 2 };

// A tile's first kilobyte, in floats.  Classes: their biases.  Rows: -maximum (powers of two), factor, label, the label's value.
constexpr int kXeShift = 0, kXeFactor = 32, kXeLabel = 64, kXeOwn = 96;

// Sizes of a problem as the kernels see it: blocks of 32 columns, padded, in one slice or two (O of one slice fits a wave's registers).
struct XeShape {
    int blocks;  // in a slice
    int slices;
    int parts;
    int cols() const { return 32 * blocks * slices; }
    int64_t s_bytes() const { return kXeChunk * (1 + 2LL * blocks * slices * parts); }  // a tile as operand of S
    int64_t p_bytes() const { return kXeChunk * 2LL * blocks * slices * parts; }        // ... of O
};

inline XeShape xe_shape(int dim, int dtype)
{
    const int n = (int)ceil_div(dim, 32);
    XeShape s;
    s.parts = dtype == FGL_F32 ? 3 : 1;
    s.slices = n > 8 ? 2 : 1;
    s.blocks = n <= 4 ? n : n <= 6 || (n > 8 && n <= 12) ? 6 : 8;
    return s;
}

// ---- images --------------------------------------------------------------------------------------------------------
struct XeMatrix {
    const void* src;
    int64_t row_stride, col_stride;  // in elements
    int64_t rows;
    char* s_image;
    char* p_image;       // or null
    const void* bias;    // classes: of the matrix's type, or null
    const void* labels;  // rows
};

struct XeImagesArgs {
    XeMatrix m[2];  // rows, classes
    int64_t first_tiles;  // of m[0]
    int dim, blocks, slices;
    int label64;
    int64_t ignore;
    int64_t classes;
};

constexpr int kXeCols = 128;  // columns that a workgroup lays out, of 32 rows
constexpr int kXePitch = kXeCols + 4;

template <int PARTS>
__device__ __forceinline__ void xe_put(const float (&v)[8], char* to)
{
    if constexpr (PARTS == 3) {
        SpU4 p[3];
        uint32_t rest = 0;  // (bits below 2^-133: nothing beside a logit, and beside a gradient of x's own size)
        sp_split(v, p, rest);
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<SpU4*>(to + q * kXeChunk) = p[q];
    } else {
        Bf16x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (__bf16)v[j];
        *reinterpret_cast<Bf16x8*>(to) = o;
    }
}

template <typename T, int PARTS>
__global__ __launch_bounds__(kBlock) void xe_images_kernel(const XeImagesArgs g)
{
    __shared__ float tile[32 * kXePitch];
    const int64_t id = blockIdx.x;
    const bool classes = id >= g.first_tiles;
    const XeMatrix& m = g.m[classes ? 1 : 0];
    const int64_t t = classes ? id - g.first_tiles : id, row0 = 32 * t;
    const int col0 = kXeCols * (int)blockIdx.y, thread = (int)threadIdx.x;
    const T* src = static_cast<const T*>(m.src);
    if (m.col_stride == 1) {
        typedef T Vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
#pragma unroll
        for (int k = 0; k < 32 * kXeCols / 8 / kBlock; ++k) {
            const int at = thread + k * kBlock, r = at / (kXeCols / 8), c = at % (kXeCols / 8) * 8, left = g.dim - col0 - c;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.0f;
            if (row0 + r < m.rows) {
                const T* p = src + (row0 + r) * m.row_stride + col0 + c;
                if (left >= 8) {
                    const Vec q = *reinterpret_cast<const Vec*>(p);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = (float)q[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < left) v[j] = (float)p[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) tile[r * kXePitch + c + j] = v[j];
        }
    } else {  // (neighbouring lanes take neighbouring rows: a transposed view's lie side by side)
#pragma unroll
        for (int k = 0; k < 32 * kXeCols / kBlock; ++k) {
            const int at = thread + k * kBlock, r = at % 32, c = at / 32;
            const bool there = row0 + r < m.rows && col0 + c < g.dim;
            tile[r * kXePitch + c] = there ? (float)src[(row0 + r) * m.row_stride + (col0 + c) * m.col_stride] : 0.0f;
        }
    }
    const int all_blocks = g.blocks * g.slices, steps = 2 * all_blocks;
    char* s_tile = m.s_image + t * kXeChunk * (1 + (int64_t)steps * PARTS);
    if (blockIdx.y == 0 && thread < 32) {
        const int64_t row = row0 + thread;
        if (classes) {
            float b = -INFINITY;
            if (row < m.rows) {
                b = m.bias != nullptr ? (float)static_cast<const T*>(m.bias)[row] : 0.0f;
                if (b <= kXeLeftOut) b = -INFINITY;
            }
            reinterpret_cast<float*>(s_tile)[thread] = b;
        } else {
            int label = -1;  // none
            if (row < m.rows) {
                const int64_t y = g.label64 ? static_cast<const int64_t*>(m.labels)[row] : (int64_t) static_cast<const int32_t*>(m.labels)[row];
                if (y != g.ignore) label = y >= 0 && y < g.classes ? (int)y : -2;  // (-2: no such class)
            }
            reinterpret_cast<int*>(s_tile)[kXeLabel + thread] = label;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int at = thread + k * kBlock, step = col0 / 16 + at / kWave, lane = at % kWave;
        if (step >= steps) break;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tile[lane % 32 * kXePitch + at / kWave * 16 + lane / 32 * 8 + j];
        xe_put<PARTS>(v, s_tile + kXeChunk * (1 + (int64_t)step * PARTS) + lane * 16);
    }
    if (m.p_image == nullptr) return;
    char* p_tile = m.p_image + t * kXeChunk * ((int64_t)steps * PARTS);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int at = thread + k * kBlock, lane = at % kWave, half = at / kWave % 2, own = at / kWave / 2, block = col0 / 32 + own;
        if (block >= all_blocks) break;
        float v[8];
        // the eight passed rows of a lane: those that its values of S^T have
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tile[(half * 16 + j / 4 * 8 + lane / 32 * 4 + j % 4) * kXePitch + own * 32 + lane % 32];
        const int slice = block / g.blocks, in_slice = block % g.blocks;
        xe_put<PARTS>(v, p_tile + kXeChunk * ((((int64_t)slice * 2 + half) * g.blocks + in_slice) * PARTS) + lane * 16);
    }
}

// ---- the passes ----------------------------------------------------------------------------------------------------
struct XeArgs {
    const char* kept;      // S images
    const char* passed;
    const char* passed_p;  // P image
    int64_t kept_tiles, passed_tiles;
    int64_t tiles_per_split;
    int splits;
    float* stats;  // [split][kept row]: maximum, others' sum, label's logit, -  (weights: sum, -, -, -)
    float* part;   // [split][slice][kept tile][block][quarter][lane][4]
    // weights without splits: straight to the result
    void* d_w;
    void* d_b;
    int64_t kept_rows;
    int dim;
    int bf16;
};

// A wave's part of a copy to LDS of `chunks` kilobytes: neither a register nor an address calculation per lane beyond the first.
template <int CHUNKS>
__device__ __forceinline__ void xe_stage(const char* src, char* dst)
{
    const int wave = (int)(threadIdx.x / kWave), lane = lane_id();
#pragma unroll
    for (int c0 = 0; c0 < CHUNKS; c0 += kXeWaves) {
        const int c = c0 + __builtin_amdgcn_readfirstlane(wave);
        if (CHUNKS % kXeWaves == 0 || c < CHUNKS)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + (int64_t)c * kXeChunk + lane * 16),
                                             (__attribute__((address_space(3))) void*)(dst + c * kXeChunk), 16, 0, 0);
    }
}

__device__ __forceinline__ void xe_staged()
{
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies have arrived
    __syncthreads();
}

__device__ __forceinline__ Bf16x8 xe_operand(const char* chunk) { return *reinterpret_cast<const Bf16x8*>(chunk + lane_id() * 16); }

__device__ __forceinline__ SpF32x16 xe_mfma(Bf16x8 a, Bf16x8 b, SpF32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

constexpr int kXePa[6] = {2, 0, 1, 1, 0, 0}, kXePb[6] = {0, 2, 1, 0, 1, 0};  // the small products first

// Waves that a SIMD (and so workgroups that a CU) holds at once: the kept rows take 8 registers a block and part, O 16 a block, of 512.
__host__ __device__ constexpr int xe_waves(int blocks, int parts, int use, bool wide)
{
    if (use == kXeLoss) return wide ? (parts == 1 ? 2 : 1) : parts == 1 ? 4 : blocks <= 2 ? 4 : blocks <= 4 ? 3 : blocks <= 6 ? 2 : 1;
    if (wide) return parts == 1 ? 2 : 1;
    return parts == 1 ? (blocks <= 2 ? 4 : blocks <= 3 ? 3 : 2) : blocks <= 1 ? 4 : blocks <= 4 ? 2 : 1;
}

template <int DB, int PARTS, int USE, bool WIDE>
struct XeWave {
    static constexpr int kSteps = WIDE ? 4 * DB : 2 * DB;
    static constexpr int kSChunks = 1 + kSteps * PARTS, kPChunks = 2 * DB * PARTS;
    static constexpr int kKept = WIDE ? 1 : kSteps;

    Bf16x8 kept[kKept][PARTS];
    const char* kept_at;  // WIDE: they are taken from memory for each tile
    SpF32x16 o[USE == kXeLoss ? 1 : DB];
    SpF32x16 start;       // weights: the class's bias sixteen times
    float top, sum, own;  // running maximum (a power of two), sum, the label's logit
    int label;            // weights: the class
    bool bias_sum;

    __device__ __forceinline__ Bf16x8 kept_part(int step, int p) const
    {
        if constexpr (WIDE) return xe_operand(kept_at + (int64_t)(step * PARTS + p) * kXeChunk);
        else return kept[step][p];
    }

    // S^T of the staged tile
    __device__ __forceinline__ SpF32x16 logits(const char* s) const
    {
        SpF32x16 acc;
        if constexpr (USE == kXeWeights) {
            acc = start;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const XeF4 b = *reinterpret_cast<const XeF4*>(s + 4 * (8 * q + 4 * (lane_id() / 32)));
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[4 * q + c] = b[c];
            }
        }
        const char* at = s + kXeChunk;
        if constexpr (PARTS == 1) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) acc = xe_mfma(xe_operand(at + k * kXeChunk), kept_part(k, 0), acc);
        } else {
#pragma unroll
            for (int k = 0; k < kSteps; k += 2) {
                SpF32x16 chunk = {};
                Bf16x8 a[2][3], b[2][3];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        a[u][p] = xe_operand(at + ((k + u) * 3 + p) * kXeChunk);
                        b[u][p] = kept_part(k + u, p);
                    }
#pragma unroll
                for (int q = 0; q < 6; ++q)
#pragma unroll
                    for (int u = 0; u < 2; ++u) chunk = xe_mfma(a[u][kXePa[q]], b[u][kXePb[q]], chunk);
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[i] += chunk[i];
            }
        }
        return acc;
    }

    // S^T -> P^T, with the running maximum, sum and the label's logit.  v0: the tile's first class.
    __device__ __forceinline__ void shares(SpF32x16& s, int64_t v0)
    {
        float most = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) most = fmaxf(most, s[i]);
        most = fmaxf(most, __shfl_xor(most, 32, kWave)) * kXeLog2e;
        if (__any(most > top + kXeStep)) {
            const float now = fmaxf(top, most);
            const float scale = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= scale;
            if constexpr (USE == kXeLossAndRows) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= scale;
            }
        }
        const float shift = top == -INFINITY ? 0.0f : -top;
        const int64_t in_tile = label - v0;
        const bool here = label >= 0 && in_tile >= 0 && in_tile < 32;
        if (__any(here)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (here && (int)in_tile == 8 * (i / 4) + 4 * (lane_id() / 32) + i % 4) {
                    own = s[i];
                    s[i] = -INFINITY;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], kXeLog2e, shift));
        add_up(s);
    }

    __device__ __forceinline__ void add_up(const SpF32x16& p)
    {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = p[i] + p[i + 8];
        sum += ((t[0] + t[4]) + (t[1] + t[5])) + ((t[2] + t[6]) + (t[3] + t[7]));
    }

    // S^T -> the gradient of the logits, from the maxima, factors and labels of the tile's rows
    __device__ __forceinline__ void gradients(SpF32x16& s, const char* tile, int64_t v0)
    {
        const float* c = reinterpret_cast<const float*>(tile);
        const int* l = reinterpret_cast<const int*>(tile);
        const int first = 4 * (lane_id() / 32);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const XeF4 shift = *reinterpret_cast<const XeF4*>(c + kXeShift + 8 * q + first), factor = *reinterpret_cast<const XeF4*>(c + kXeFactor + 8 * q + first);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[4 * q + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * q + j], kXeLog2e, shift[j])) * factor[j];
        }
        const int64_t in_tile = l[kXeLabel + lane_id() % 32] - v0;
        if (__any(in_tile >= 0 && in_tile < 32)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int n = 8 * (i / 4) + first + i % 4;
                if (l[kXeLabel + n] == label) s[i] = c[kXeOwn + n];
            }
        }
        if (bias_sum) add_up(s);
    }

    // O^T += passed^T P^T
    __device__ __forceinline__ void product(const SpF32x16& s, const char* p)
    {
        if constexpr (PARTS == 1) {
            Bf16x8 w[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i / 8][i % 8] = (__bf16)s[i];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = xe_mfma(xe_operand(p + (h * DB + d) * kXeChunk), w[h], o[d]);
        } else {
            SpU4 w[2][3];
            uint32_t rest = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = s[8 * h + j];
                sp_split(v, w[h], rest);
            }
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                SpF32x16 chunk = {};
                Bf16x8 a[2][3];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < 3; ++q) a[h][q] = xe_operand(p + ((h * DB + d) * 3 + q) * kXeChunk);
#pragma unroll
                for (int q = 0; q < 6; ++q)
#pragma unroll
                    for (int h = 0; h < 2; ++h) chunk = xe_mfma(a[h][kXePa[q]], __builtin_bit_cast(Bf16x8, w[h][kXePb[q]]), chunk);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] += chunk[i];
            }
        }
    }

    // One tile: copies what comes next to `next` while it works on `s`
    __device__ __forceinline__ void first_half(const char* __restrict__ s, char* __restrict__ next, const char* src, SpF32x16& p, int64_t n0, int64_t v0, bool active)
    {
        if constexpr (USE == kXeLoss) {
            if (src != nullptr) xe_stage<kSChunks>(src, next);
        } else {
            xe_stage<kPChunks>(src, next);
        }
        if (!active) return;
        p = logits(s);
        if constexpr (USE == kXeWeights) gradients(p, s, v0);
        else shares(p, n0);
    }
    __device__ __forceinline__ void second_half(const char* __restrict__ s, char* __restrict__ next, const char* src, const SpF32x16& p, bool active)
    {
        if (src != nullptr) xe_stage<kSChunks>(src, next);
        if (active) product(p, s);
    }
};

template <int DB, int PARTS, int USE, bool WIDE>
__global__ __launch_bounds__(kBlock, xe_waves(DB, PARTS, USE, WIDE)) void xe_kernel(const XeArgs g)
{
    using Wave = XeWave<DB, PARTS, USE, WIDE>;
    // the loss alone: two tiles in turn, or one where LDS has no room for two
    constexpr bool kTwo = USE == kXeLoss && 2 * Wave::kSChunks <= 160;
    __shared__ __attribute__((aligned(16))) char s_buf[Wave::kSChunks * kXeChunk];
    __shared__ __attribute__((aligned(16))) char p_buf[(USE != kXeLoss ? Wave::kPChunks : kTwo ? Wave::kSChunks : 1) * kXeChunk];
    constexpr int kSlices = WIDE && USE != kXeLoss ? 2 : 1;
    constexpr int64_t kSBytes = (int64_t)Wave::kSChunks * kXeChunk, kPBytes = (int64_t)Wave::kPChunks * (WIDE ? 2 : 1) * kXeChunk;
    const int split = (int)(blockIdx.x % (unsigned)g.splits);
    const int rest = (int)(blockIdx.x / (unsigned)g.splits), slice = rest % kSlices;
    const int lane = lane_id();
    const int64_t tile = (int64_t)(rest / kSlices) * kXeWaves + __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const bool active = tile < g.kept_tiles;
    const int64_t mine = active ? tile : g.kept_tiles - 1;
    const char* own = g.kept + mine * kSBytes;

    Wave w;
    w.kept_at = own + kXeChunk;
    if constexpr (!WIDE) {
#pragma unroll
        for (int k = 0; k < Wave::kSteps; ++k)
#pragma unroll
            for (int p = 0; p < PARTS; ++p) w.kept[k][p] = xe_operand(w.kept_at + (k * PARTS + p) * kXeChunk);
    }
#pragma unroll
    for (int d = 0; d < (USE == kXeLoss ? 1 : DB); ++d) w.o[d] = SpF32x16{};
    w.top = -INFINITY;
    w.sum = w.own = 0.0f;
    w.bias_sum = g.d_b != nullptr;
    if constexpr (USE == kXeWeights) {
        w.label = (int)(32 * tile) + lane % 32;
        const float b = reinterpret_cast<const float*>(own)[lane % 32];
#pragma unroll
        for (int i = 0; i < 16; ++i) w.start[i] = b;
    } else {
        w.label = reinterpret_cast<const int*>(own)[kXeLabel + lane % 32];
    }

    const int64_t t0 = split * g.tiles_per_split, t1 = t0 + g.tiles_per_split < g.passed_tiles ? t0 + g.tiles_per_split : g.passed_tiles;
    const int64_t v0 = 32 * tile;
    SpF32x16 p = {};
    xe_stage<Wave::kSChunks>(g.passed + t0 * kSBytes, s_buf);
    xe_staged();
    if constexpr (USE == kXeLoss && !kTwo) {
        for (int64_t t = t0; t < t1; ++t) {
            w.first_half(s_buf, p_buf, nullptr, p, 32 * t, v0, active);
            __syncthreads();
            if (t + 1 < t1) xe_stage<Wave::kSChunks>(g.passed + (t + 1) * kSBytes, s_buf);
            xe_staged();
        }
    } else if constexpr (USE == kXeLoss) {
        for (int64_t t = t0; t < t1; t += 2) {
            w.first_half(s_buf, p_buf, t + 1 < t1 ? g.passed + (t + 1) * kSBytes : nullptr, p, 32 * t, v0, active);
            xe_staged();
            if (t + 1 == t1) break;
            w.first_half(p_buf, s_buf, t + 2 < t1 ? g.passed + (t + 2) * kSBytes : nullptr, p, 32 * (t + 1), v0, active);
            xe_staged();
        }
    } else {
        const char* passed_p = g.passed_p + slice * (int64_t)Wave::kPChunks * kXeChunk;
        for (int64_t t = t0; t < t1; ++t) {
            w.first_half(s_buf, p_buf, passed_p + t * kPBytes, p, 32 * t, v0, active);
            xe_staged();
            w.second_half(p_buf, s_buf, t + 1 < t1 ? g.passed + (t + 1) * kSBytes : nullptr, p, active);
            xe_staged();
        }
    }
    if (!active) return;

    w.sum += __shfl_xor(w.sum, 32, kWave);
    w.own += __shfl_xor(w.own, 32, kWave);
    const int half = lane / 32;
    if constexpr (USE == kXeWeights) {
        if (g.splits == 1) {
            const int64_t row = v0 + lane % 32;
            if (row >= g.kept_rows) return;
            if (g.d_b != nullptr && half == 0 && slice == 0) {
                if (g.bf16) static_cast<__bf16*>(g.d_b)[row] = (__bf16)w.sum;
                else static_cast<float*>(g.d_b)[row] = w.sum;
            }
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int col = 32 * (slice * DB + d) + 8 * q + 4 * half;
                    const int64_t to = row * g.dim + col;
                    float v[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[c] = w.o[d][4 * q + c];
                    if (g.bf16) {
                        typedef __bf16 Vec __attribute__((ext_vector_type(4), aligned(2)));
                        __bf16* out = static_cast<__bf16*>(g.d_w) + to;
                        if (col + 4 <= g.dim) *reinterpret_cast<Vec*>(out) = Vec{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
                        else
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (col + c < g.dim) out[c] = (__bf16)v[c];
                    } else {
                        typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
                        float* out = static_cast<float*>(g.d_w) + to;
                        if (col + 4 <= g.dim) *reinterpret_cast<Vec*>(out) = Vec{v[0], v[1], v[2], v[3]};
                        else
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (col + c < g.dim) out[c] = v[c];
                    }
                }
            return;
        }
    }
    if (half == 0 && slice == 0) {
        const XeF4 v = USE == kXeWeights ? XeF4{w.sum, 0.0f, 0.0f, 0.0f} : XeF4{w.top, w.sum, w.own, 0.0f};
        *reinterpret_cast<XeF4*>(g.stats + 4 * (split * 32 * g.kept_tiles + v0 + lane)) = v;
    }
    if constexpr (USE != kXeLoss) {
        float* to = g.part + (((int64_t)split * kSlices + slice) * g.kept_tiles + tile) * (DB * 4 * kWave * 4) + lane * 4;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<XeF4*>(to + (d * 4 + q) * kWave * 4) = XeF4{w.o[d][4 * q], w.o[d][4 * q + 1], w.o[d][4 * q + 2], w.o[d][4 * q + 3]};
    }
}

// ---- what the splits left, added up --------------------------------------------------------------------------------
struct XeRow {  // of a row, for the backward pass
    float top, inverse, others;  // maximum (a power of two), 1 / sum, the other classes' share
    int label;
};

struct XeCombineArgs {
    const float* stats;
    const float* part;
    const char* rows;  // S image of the rows (labels)
    int64_t tiles, n_rows, s_bytes;
    int splits, blocks, slices;
    const void* w;  // classes
    int64_t w_row, w_col;
    int dim, bf16;
    float* losses;     // a row each, or null
    float* tile_loss;  // [tile][2]: sum, count
    XeRow* kept;       // or null
    float* d_x;        // [row][padded columns], up to its factor, or null
};

// (one workgroup a tile of 32 rows)
__global__ __launch_bounds__(kBlock) void xe_combine_kernel(const XeCombineArgs g)
{
    __shared__ float scale[kXeMaxSplits * 32];
    __shared__ float others[32];
    __shared__ int labels[32];
    const int64_t tile = blockIdx.x, row0 = 32 * tile;
    const int thread = (int)threadIdx.x;
    if (thread < kWave) {
        const int i = thread % 32;
        const bool there = row0 + i < g.n_rows;
        const int label = reinterpret_cast<const int*>(g.rows + tile * g.s_bytes)[kXeLabel + i];
        const XeF4* s = reinterpret_cast<const XeF4*>(g.stats) + row0 + i;
        const int64_t step = 32 * g.tiles;
        float top = -INFINITY, own = 0.0f;
        for (int k = 0; k < g.splits; ++k) {
            const XeF4 v = s[k * step];
            top = fmaxf(top, v[0]);
            own += v[2];
        }
        const float own2 = own * kXeLog2e;
        if (label >= 0) top = fmaxf(top, own2);
        float rest = 0.0f;
        for (int k = 0; k < g.splits; ++k) {
            const XeF4 v = s[k * step];
            const float f = v[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v[0] - top);
            rest += v[0] == -INFINITY ? v[1] : v[1] * f;  // (what is not a number stays it)
            if (thread < 32) scale[k * 32 + i] = f;
        }
        const float mine = label >= 0 ? __builtin_amdgcn_exp2f(own2 - top) : 0.0f;
        const float total = rest + mine, inverse = 1.0f / total;
        float loss = top - own2 < 64.0f ? log1pf(rest / mine) : kXeLn2 * top + logf(total) - own;
        float share = rest * inverse;
        if (label == -2) loss = share = NAN;
        if (label == -1) loss = share = 0.0f;
        if (thread < 32) {
            if (there) {
                if (g.losses != nullptr) g.losses[row0 + i] = loss;
                if (g.kept != nullptr) g.kept[row0 + i] = XeRow{top, inverse, share, label};
            }
            others[i] = share;
            labels[i] = there ? label : -1;
            for (int k = 0; k < g.splits; ++k) scale[k * 32 + i] *= inverse;
        }
        float sum = there && thread < 32 ? loss : 0.0f, count = there && thread < 32 && label != -1 ? 1.0f : 0.0f;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) {
            sum += __shfl_xor(sum, d, kWave);
            count += __shfl_xor(count, d, kWave);
        }
        if (thread == 0 && g.tile_loss != nullptr) {
            g.tile_loss[2 * tile] = sum;
            g.tile_loss[2 * tile + 1] = count;
        }
    }
    if (g.d_x == nullptr) return;
    __syncthreads();
    const int cols = 32 * g.blocks * g.slices, per_slice = g.blocks * 4 * kWave;
    const int64_t slice_step = g.tiles * per_slice;
    for (int at = thread; at < per_slice * g.slices; at += kBlock) {
        const int slice = at / per_slice, in_slice = at % per_slice, lane = in_slice % kWave, i = lane % 32;
        const int col = 32 * (slice * g.blocks) + in_slice / kWave * 8 + lane / 32 * 4;
        if (row0 + i >= g.n_rows) continue;
        const XeF4* p = reinterpret_cast<const XeF4*>(g.part) + (slice * g.tiles + tile) * per_slice + in_slice;
        XeF4 sum = {};
        for (int k = 0; k < g.splits; ++k) {
            const XeF4 v = p[k * g.slices * slice_step];
            const float f = scale[k * 32 + i];
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += v[c] * f;
        }
        const int label = labels[i];
        if (label >= 0) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (col + c >= g.dim) continue;
                const int64_t from = label * g.w_row + (col + c) * g.w_col;
                const float v = g.bf16 ? (float)static_cast<const __bf16*>(g.w)[from] : static_cast<const float*>(g.w)[from];
                sum[c] -= others[i] * v;
            }
        }
        *reinterpret_cast<XeF4*>(g.d_x + (row0 + i) * cols + col) = sum;
    }
}

// the tiles' losses -> *loss; *count: rows with a label
__global__ __launch_bounds__(kBlock) void xe_total_kernel(const float* __restrict__ tile_loss, int64_t tiles, int mean, float* __restrict__ loss, float* __restrict__ count)
{
    __shared__ double s[kBlock], c[kBlock];
    double sum = 0.0, n = 0.0;
    for (int64_t t = threadIdx.x; t < tiles; t += kBlock) {
        sum += (double)tile_loss[2 * t];
        n += (double)tile_loss[2 * t + 1];
    }
    s[threadIdx.x] = sum;
    c[threadIdx.x] = n;
    __syncthreads();
    for (int d = kBlock / 2; d >= 1; d >>= 1) {
        if ((int)threadIdx.x < d) {
            s[threadIdx.x] += s[threadIdx.x + d];
            c[threadIdx.x] += c[threadIdx.x + d];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *loss = (float)(mean ? s[0] / c[0] : s[0]);  // (no labels at all: not a number, as the mean of nothing is)
        *count = (float)c[0];
    }
}

struct XeRowsArgs {
    const XeRow* kept;
    const float* d_x;  // or null
    const float* d_loss;
    const float* count;
    int reduction;
    char* rows;  // S image of the rows, or null: the factors of the weights' gradient
    int64_t tiles, n_rows, s_bytes;
    int cols, dim, bf16;
    void* out;
};

// The factors of a tile's 32 rows, and dx from them.
__global__ __launch_bounds__(kBlock) void xe_rows_kernel(const XeRowsArgs g)
{
    __shared__ float factor[32];
    __shared__ int labels[32];
    const int64_t tile = blockIdx.x, row0 = 32 * tile;
    const int thread = (int)threadIdx.x;
    if (thread < 32) {
        const bool there = row0 + thread < g.n_rows;
        const XeRow r = there ? g.kept[row0 + thread] : XeRow{0.0f, 0.0f, 0.0f, -1};
        float f = 0.0f;
        if (there) f = g.reduction == FGL_REDUCE_NONE ? g.d_loss[row0 + thread] : g.reduction == FGL_REDUCE_SUM ? *g.d_loss : *g.d_loss / *g.count;
        const bool with = r.label != -1;
        factor[thread] = r.label == -2 ? NAN : f;
        labels[thread] = r.label;
        if (g.rows != nullptr) {
            float* c = reinterpret_cast<float*>(g.rows + tile * g.s_bytes);
            c[kXeShift + thread] = with ? (r.label == -2 ? NAN : -r.top) : -INFINITY;
            c[kXeFactor + thread] = with ? f * r.inverse : 0.0f;
            c[kXeOwn + thread] = -f * r.others;
        }
    }
    if (g.out == nullptr) return;
    __syncthreads();
    const int quads = (g.dim + 3) / 4;
    for (int at = thread; at < 32 * quads; at += kBlock) {
        const int i = at / quads, col = at % quads * 4;
        if (row0 + i >= g.n_rows) break;
        XeF4 v = *reinterpret_cast<const XeF4*>(g.d_x + (row0 + i) * g.cols + col);
        const bool with = labels[i] != -1;
        const int64_t to = (row0 + i) * g.dim + col;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (col + c >= g.dim) continue;
            const float d = with ? v[c] * factor[i] : 0.0f;
            if (g.bf16) static_cast<__bf16*>(g.out)[to + c] = (__bf16)d;
            else static_cast<float*>(g.out)[to + c] = d;
        }
    }
}

struct XeWeightsArgs {
    const float* stats;
    const float* part;
    int64_t tiles, n_rows;
    int splits, blocks, slices, dim, bf16;
    void* d_w;
    void* d_b;  // or null
};

__global__ __launch_bounds__(kBlock) void xe_weights_kernel(const XeWeightsArgs g)
{
    const int64_t tile = blockIdx.x, row0 = 32 * tile;
    const int thread = (int)threadIdx.x;
    if (g.d_b != nullptr && thread < 32 && row0 + thread < g.n_rows && blockIdx.y == 0) {
        float sum = 0.0f;
        for (int k = 0; k < g.splits; ++k) sum += g.stats[4 * (k * 32 * g.tiles + row0 + thread)];
        if (g.bf16) static_cast<__bf16*>(g.d_b)[row0 + thread] = (__bf16)sum;
        else static_cast<float*>(g.d_b)[row0 + thread] = sum;
    }
    const int per_slice = g.blocks * 4 * kWave;
    const int64_t slice_step = g.tiles * per_slice;
    for (int at = (int)blockIdx.y * kBlock + thread; at < per_slice * g.slices; at += kBlock * (int)gridDim.y) {
        const int slice = at / per_slice, in_slice = at % per_slice, lane = in_slice % kWave, i = lane % 32;
        const int col = 32 * (slice * g.blocks) + in_slice / kWave * 8 + lane / 32 * 4;
        if (row0 + i >= g.n_rows || col >= g.dim) continue;
        const XeF4* p = reinterpret_cast<const XeF4*>(g.part) + (slice * g.tiles + tile) * per_slice + in_slice;
        XeF4 sum = {};
        for (int k = 0; k < g.splits; ++k) {
            const XeF4 v = p[k * g.slices * slice_step];
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += v[c];
        }
        const int64_t to = (row0 + i) * g.dim + col;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (col + c >= g.dim) continue;
            if (g.bf16) static_cast<__bf16*>(g.d_w)[to + c] = (__bf16)sum[c];
            else static_cast<float*>(g.d_w)[to + c] = sum[c];
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------
struct XeSplit {
    int splits;
    int64_t tiles;  // of each
};

inline XeSplit xe_split(const XeShape& s, int use, int64_t kept_tiles, int64_t passed_tiles)
{
    const int64_t groups = ceil_div(kept_tiles, kXeWaves) * (use == kXeLoss ? 1 : s.slices);
    int64_t n = 256LL * xe_waves(s.blocks, s.parts, use, s.slices == 2) / groups;
    if (n > kXeMaxSplits) n = kXeMaxSplits;
    if (n > passed_tiles) n = passed_tiles;
    if (n < 1) n = 1;
    XeSplit r;
    r.tiles = ceil_div(passed_tiles, n);
    r.splits = (int)ceil_div(passed_tiles, r.tiles);
    return r;
}

struct XeProblem {
    int64_t n, classes, row_tiles, class_tiles;
    int dim, dtype;
    XeShape shape;
};

inline bool xe_problem(int64_t n, int64_t classes, int dim, int dtype, XeProblem* p)
{
    if (n < 1 || n >= (1LL << 31) - 64 || classes < 1 || classes >= (1LL << 31) - 64 || dim < 1 || dim > kXeMaxDim || (dtype != FGL_F32 && dtype != FGL_BF16)) return false;
    p->n = n;
    p->classes = classes;
    p->dim = dim;
    p->dtype = dtype;
    p->row_tiles = ceil_div(n, 32);
    p->class_tiles = ceil_div(classes, 32);
    p->shape = xe_shape(dim, dtype);
    return true;
}

// What a forward pass leaves for the backward one, and its scratch.
struct XeState {
    char *rows_s, *rows_p, *classes_s;  // (weights' gradient)
    XeRow* kept;
    float* d_x;
    float* count;
    size_t bytes;
};

inline XeState xe_state(const XeProblem& p, int want, void* base)
{
    Carver c(base);
    XeState s = {};
    s.count = c.take<float>(1);
    if (want != 0) s.kept = c.take<XeRow>((size_t)p.n);
    if (want & FGL_XENT_ROWS) s.d_x = c.take<float>((size_t)p.n * p.shape.cols());
    if (want & FGL_XENT_WEIGHTS) {
        s.rows_s = c.take<char>((size_t)(p.row_tiles * p.shape.s_bytes()));
        s.rows_p = c.take<char>((size_t)(p.row_tiles * p.shape.p_bytes()));
        s.classes_s = c.take<char>((size_t)(p.class_tiles * p.shape.s_bytes()));
    }
    s.bytes = c.used();
    return s;
}

struct XeScratch {
    char *rows_s, *classes_s, *classes_p;
    float *stats, *part, *tile_loss;
    size_t bytes;
};

inline XeScratch xe_forward_scratch(const XeProblem& p, int want, void* base)
{
    const int use = want & FGL_XENT_ROWS ? kXeLossAndRows : kXeLoss;
    const XeSplit split = xe_split(p.shape, use, p.row_tiles, p.class_tiles);
    Carver c(base);
    XeScratch s = {};
    if (!(want & FGL_XENT_WEIGHTS)) {
        s.rows_s = c.take<char>((size_t)(p.row_tiles * p.shape.s_bytes()));
        s.classes_s = c.take<char>((size_t)(p.class_tiles * p.shape.s_bytes()));
    }
    if (use == kXeLossAndRows) {
        s.classes_p = c.take<char>((size_t)(p.class_tiles * p.shape.p_bytes()));
        s.part = c.take<float>((size_t)(split.splits * p.row_tiles) * 32 * p.shape.cols());
    }
    s.stats = c.take<float>((size_t)split.splits * p.row_tiles * 32 * 4);
    s.tile_loss = c.take<float>((size_t)p.row_tiles * 2);
    s.bytes = c.used();
    return s;
}

inline XeScratch xe_backward_scratch(const XeProblem& p, int want, void* base)
{
    Carver c(base);
    XeScratch s = {};
    if (want & FGL_XENT_WEIGHTS) {
        const XeSplit split = xe_split(p.shape, kXeWeights, p.class_tiles, p.row_tiles);
        if (split.splits > 1) {
            s.part = c.take<float>((size_t)(split.splits * p.class_tiles) * 32 * p.shape.cols());
            s.stats = c.take<float>((size_t)split.splits * p.class_tiles * 32 * 4);
        }
    }
    s.bytes = c.used();
    return s;
}

template <int PARTS, int USE>
void launch_xe_parts(const XeShape& s, const XeArgs& g, unsigned groups, hipStream_t stream)
{
    const dim3 grid(groups), block(kBlock);
    if (s.slices == 2) {
        if (s.blocks == 6) hipLaunchKernelGGL((xe_kernel<6, PARTS, USE, true>), grid, block, 0, stream, g);
        else hipLaunchKernelGGL((xe_kernel<8, PARTS, USE, true>), grid, block, 0, stream, g);
        return;
    }
    switch (s.blocks) {
    case 1: hipLaunchKernelGGL((xe_kernel<1, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 2: hipLaunchKernelGGL((xe_kernel<2, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 3: hipLaunchKernelGGL((xe_kernel<3, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 4: hipLaunchKernelGGL((xe_kernel<4, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 6: hipLaunchKernelGGL((xe_kernel<6, PARTS, USE, false>), grid, block, 0, stream, g); break;
    default: hipLaunchKernelGGL((xe_kernel<8, PARTS, USE, false>), grid, block, 0, stream, g); break;
    }
}

template <int USE>
int launch_xe(const XeShape& s, XeArgs& g, hipStream_t stream)
{
    const XeSplit split = xe_split(s, USE, g.kept_tiles, g.passed_tiles);
    g.splits = split.splits;
    g.tiles_per_split = split.tiles;
    const int64_t groups = ceil_div(g.kept_tiles, kXeWaves) * (USE == kXeLoss ? 1 : s.slices) * split.splits;
    if (groups >= 1 << 24) {
        set_error("linear_cross_entropy: grid too large");
        return FGL_ERR_UNSUPPORTED;
    }
    if (s.parts == 3) launch_xe_parts<3, USE>(s, g, (unsigned)groups, stream);
    else launch_xe_parts<1, USE>(s, g, (unsigned)groups, stream);
    return FGL_OK;
}

}  // namespace fgl

using namespace fgl;

FGL_EXPORT size_t fgl_linear_cross_entropy_state_bytes(int64_t n_rows, int64_t n_classes, int dim, int dtype, int want)
{
    XeProblem p;
    return xe_problem(n_rows, n_classes, dim, dtype, &p) ? xe_state(p, want, nullptr).bytes : 0;
}

FGL_EXPORT size_t fgl_linear_cross_entropy_workspace_bytes(int64_t n_rows, int64_t n_classes, int dim, int dtype, int want, int backward)
{
    XeProblem p;
    if (!xe_problem(n_rows, n_classes, dim, dtype, &p)) return 0;
    return backward ? xe_backward_scratch(p, want, nullptr).bytes : xe_forward_scratch(p, want, nullptr).bytes;
}

FGL_EXPORT int fgl_linear_cross_entropy(const void* d_x, int64_t x_row_stride, int64_t x_col_stride, const void* d_w, int64_t w_row_stride, int64_t w_col_stride,
                                        const void* d_bias, const void* d_labels, int label64, int64_t ignore_index, int64_t n_rows, int64_t n_classes, int dim,
                                        int dtype, int reduction, int want, float* d_loss, void* d_state, size_t state_bytes, void* d_ws, size_t ws_bytes,
                                        void* stream)
{
    XeProblem p;
    FGL_REQUIRE(xe_problem(n_rows, n_classes, dim, dtype, &p), "linear_cross_entropy: %lld rows and %lld classes of %d columns (1 .. %d), dtype %d",
                (long long)n_rows, (long long)n_classes, dim, kXeMaxDim, dtype);
    FGL_REQUIRE(reduction == FGL_REDUCE_NONE || reduction == FGL_REDUCE_SUM || reduction == FGL_REDUCE_MEAN, "linear_cross_entropy: reduction %d", reduction);
    FGL_REQUIRE((want & ~(FGL_XENT_ROWS | FGL_XENT_WEIGHTS)) == 0, "linear_cross_entropy: want %d", want);
    FGL_REQUIRE(d_x && d_w && d_labels && d_loss && d_state && d_ws, "linear_cross_entropy: null pointer");
    const XeState st = xe_state(p, want, d_state);
    const XeScratch ws = xe_forward_scratch(p, want, d_ws);
    if (state_bytes < st.bytes || ws_bytes < ws.bytes || ((uintptr_t)d_state | (uintptr_t)d_ws) % 256 != 0) {
        set_error("linear_cross_entropy: needs %zu bytes of state and %zu of workspace on 256-byte boundaries, got %zu and %zu", st.bytes, ws.bytes, state_bytes, ws_bytes);
        return FGL_ERR_WORKSPACE;
    }
    const XeShape& s = p.shape;
    const hipStream_t to = as_stream(stream);
    XeImagesArgs im = {};
    im.m[0] = XeMatrix{d_x, x_row_stride, x_col_stride, n_rows, st.rows_s ? st.rows_s : ws.rows_s, st.rows_p, nullptr, d_labels};
    im.m[1] = XeMatrix{d_w, w_row_stride, w_col_stride, n_classes, st.classes_s ? st.classes_s : ws.classes_s, ws.classes_p, d_bias, nullptr};
    im.first_tiles = p.row_tiles;
    im.dim = dim;
    im.blocks = s.blocks;
    im.slices = s.slices;
    im.label64 = label64;
    im.ignore = ignore_index;
    im.classes = n_classes;
    const int64_t tiles = p.row_tiles + p.class_tiles;
    FGL_REQUIRE(tiles < 1 << 24, "linear_cross_entropy: grid too large");
    const dim3 grid((unsigned)tiles, (unsigned)ceil_div(s.cols(), kXeCols)), block(kBlock);
    if (dtype == FGL_F32) hipLaunchKernelGGL((xe_images_kernel<float, 3>), grid, block, 0, to, im);
    else hipLaunchKernelGGL((xe_images_kernel<__bf16, 1>), grid, block, 0, to, im);
    FGL_CHECK_LAUNCH("xe_images_kernel");

    XeArgs g = {};
    g.kept = im.m[0].s_image;
    g.passed = im.m[1].s_image;
    g.passed_p = ws.classes_p;
    g.kept_tiles = p.row_tiles;
    g.passed_tiles = p.class_tiles;
    g.stats = ws.stats;
    g.part = ws.part;
    const int rc = want & FGL_XENT_ROWS ? launch_xe<kXeLossAndRows>(s, g, to) : launch_xe<kXeLoss>(s, g, to);
    if (rc != FGL_OK) return rc;
    FGL_CHECK_LAUNCH("xe_kernel");

    XeCombineArgs c = {};
    c.stats = ws.stats;
    c.part = ws.part;
    c.rows = g.kept;
    c.tiles = p.row_tiles;
    c.n_rows = n_rows;
    c.s_bytes = s.s_bytes();
    c.splits = g.splits;
    c.blocks = s.blocks;
    c.slices = s.slices;
    c.w = d_w;
    c.w_row = w_row_stride;
    c.w_col = w_col_stride;
    c.dim = dim;
    c.bf16 = dtype == FGL_BF16;
    c.losses = reduction == FGL_REDUCE_NONE ? d_loss : nullptr;
    c.tile_loss = reduction == FGL_REDUCE_NONE ? nullptr : ws.tile_loss;
    c.kept = st.kept;
    c.d_x = st.d_x;
    hipLaunchKernelGGL(xe_combine_kernel, dim3((unsigned)p.row_tiles), block, 0, to, c);
    FGL_CHECK_LAUNCH("xe_combine_kernel");
    if (reduction != FGL_REDUCE_NONE) {
        hipLaunchKernelGGL(xe_total_kernel, dim3(1), block, 0, to, ws.tile_loss, p.row_tiles, (int)(reduction == FGL_REDUCE_MEAN), d_loss, st.count);
        FGL_CHECK_LAUNCH("xe_total_kernel");
    }
    return FGL_OK;
}

FGL_EXPORT int fgl_linear_cross_entropy_backward(const float* d_loss_grad, int64_t n_rows, int64_t n_classes, int dim, int dtype, int reduction, int want,
                                                 void* d_state, size_t state_bytes, void* d_dx, void* d_dw, void* d_db, void* d_ws, size_t ws_bytes, void* stream)
{
    XeProblem p;
    FGL_REQUIRE(xe_problem(n_rows, n_classes, dim, dtype, &p), "linear_cross_entropy_backward: %lld rows and %lld classes of %d columns (1 .. %d), dtype %d",
                (long long)n_rows, (long long)n_classes, dim, kXeMaxDim, dtype);
    FGL_REQUIRE(reduction == FGL_REDUCE_NONE || reduction == FGL_REDUCE_SUM || reduction == FGL_REDUCE_MEAN, "linear_cross_entropy_backward: reduction %d", reduction);
    FGL_REQUIRE((want & ~(FGL_XENT_ROWS | FGL_XENT_WEIGHTS)) == 0 && want != 0, "linear_cross_entropy_backward: want %d", want);
    FGL_REQUIRE(d_loss_grad && d_state && d_ws && (d_dx == nullptr || (want & FGL_XENT_ROWS)) && ((d_dw == nullptr && d_db == nullptr) || (want & FGL_XENT_WEIGHTS)) &&
                    (d_db == nullptr || d_dw != nullptr),
                "linear_cross_entropy_backward: null pointer, or a gradient that the forward pass was not told of");
    const XeState st = xe_state(p, want, d_state);
    const XeScratch ws = xe_backward_scratch(p, want, d_ws);
    if (state_bytes < st.bytes || ws_bytes < ws.bytes || ((uintptr_t)d_state | (uintptr_t)d_ws) % 256 != 0) {
        set_error("linear_cross_entropy_backward: needs %zu bytes of state and %zu of workspace on 256-byte boundaries, got %zu and %zu", st.bytes, ws.bytes, state_bytes, ws_bytes);
        return FGL_ERR_WORKSPACE;
    }
    const XeShape& s = p.shape;
    const hipStream_t to = as_stream(stream);
    const dim3 block(kBlock);
    XeRowsArgs r = {};
    r.kept = st.kept;
    r.d_x = st.d_x;
    r.d_loss = d_loss_grad;
    r.count = st.count;
    r.reduction = reduction;
    r.rows = d_dw != nullptr ? st.rows_s : nullptr;
    r.tiles = p.row_tiles;
    r.n_rows = n_rows;
    r.s_bytes = s.s_bytes();
    r.cols = s.cols();
    r.dim = dim;
    r.bf16 = dtype == FGL_BF16;
    r.out = d_dx;
    hipLaunchKernelGGL(xe_rows_kernel, dim3((unsigned)p.row_tiles), block, 0, to, r);
    FGL_CHECK_LAUNCH("xe_rows_kernel");
    if (d_dw == nullptr) return FGL_OK;

    XeArgs g = {};
    g.kept = st.classes_s;
    g.passed = st.rows_s;
    g.passed_p = st.rows_p;
    g.kept_tiles = p.class_tiles;
    g.passed_tiles = p.row_tiles;
    g.stats = ws.stats;
    g.part = ws.part;
    g.d_w = d_dw;
    g.d_b = d_db;
    g.kept_rows = n_classes;
    g.dim = dim;
    g.bf16 = dtype == FGL_BF16;
    const int rc = launch_xe<kXeWeights>(s, g, to);
    if (rc != FGL_OK) return rc;
    FGL_CHECK_LAUNCH("xe_kernel");
    if (g.splits > 1) {
        XeWeightsArgs c = {};
        c.stats = ws.stats;
        c.part = ws.part;
        c.tiles = p.class_tiles;
        c.n_rows = n_classes;
        c.splits = g.splits;
        c.blocks = s.blocks;
        c.slices = s.slices;
        c.dim = dim;
        c.bf16 = g.bf16;
        c.d_w = d_dw;
        c.d_b = d_db;
        hipLaunchKernelGGL(xe_weights_kernel, dim3((unsigned)p.class_tiles, (unsigned)s.blocks), block, 0, to, c);
        FGL_CHECK_LAUNCH("xe_weights_kernel");
    }
    return FGL_OK;
}
