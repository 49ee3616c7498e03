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
// The running maximum is moved only where a row's largest value passes it by 2^8, so that O is rescaled a few times a pass and not once a
// tile.  The label's own share is no part of maximum, sum and O.
//
// Operands: "images" (xe_images_kernel), a copy of x and w in the order in which the lanes take them, 1 KB for each 32 x 16 values, rows
// and columns padded with zeros: once as operand of S (lane: row, eight columns) and once of O (lane: column, eight rows).  So a tile is
// copied to LDS straight, without a register or a bank conflict, and no access is out of bounds whatever the sizes.  A tile's
// first kilobyte has what belongs to its 32 rows: biases, or labels and the backward pass's factors.
//
// bf16: P is rounded to bf16, as the operands are.
// fp32: each value, P's and the logits' gradients' among them, is the sum of three bf16 values, exactly (fgl_split.hpp), and a product six matrix
// instructions, the small ones first, that add to fp32 accumulators; what is left out is 2^-23 of the product at most.  So each term of a sum has
// fp32's precision for itself, however far rows, columns and classes lie apart.  (Two fp16 parts and three instructions a product take
// two thirds of the time, 8192 x 128, 20 K classes, forward and backward 498 us for 782, but share a power of two with the values around them and
// hold nothing below 2^-39 of the largest of those: one column of x 2^30 times the others took half of the other columns' bits.)
// Sums, maxima and losses are fp32 in both.  x and w must be finite, and below 3.38e38 in fp32, where a part would round to infinity: others make
// losses and gradients that are not numbers, but in rows without a label and in classes that are left out, which are taken as zeros.
// A bias of -1e30 or less, -infinity among them, leaves its class out: no share, no gradient.  (Shares are exp2 of one fma, whose
// product with log2 e is not rounded where the maximum's is: logits up to some 1e9 are no matter, the difference of 2^-25 of the maximum is the
// same for all of a row's shares and their sum.)
//
// Work: four kept tiles (a group, one a wave) times the passed tiles, dealt out to as many workgroups as the chip holds (XePlan): a group is shared by
// several, each with a part of the passed tiles, or a workgroup goes on from one group to the next in the middle of it.  Who has but a
// part of a group's tiles leaves its O, maximum and sum in scratch, and a combining kernel adds the parts up in order (the same bits on every
// run).
//
// What bounds it: for many classes the matrix cores and, beside them, LDS, whose operands at 1 KB for an instruction of 32 cycles would take all of its
// rate if the cores were never idle.  8192 x 256, 100 K classes, bf16: 690 .. 770 us forward, 735 .. 835 backward (the clock falls as the chip warms up),
// 1.00 .. 1.22 PFLOP/s (a large matrix product of the library 1.24), matrix cores busy 63 and 57 % of the cycles at the 1.8 GHz that the power limit
// leaves.  8192 x 128, 20 K classes, fp32: 372 .. 397 us and 386 .. 419, 1.20 .. 1.35 PFLOP/s of bf16 (six products), busy 68 and 64 % beside the exponentials and splits.
// The loss alone, bf16, is bound by the exponentials, maxima and sums: 2000 x 100, 100 K classes 66 us, busy 34 %.  For a few classes: launches of 5 to
// 20 us, mostly latency.
#include "fgl_common.hpp"
#include "fgl_kernels.hpp"
#include "fgl_split.hpp"

#include <math.h>

#include <type_traits>

namespace fgl {

typedef float XeF4 __attribute__((ext_vector_type(4)));
typedef float XeF32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t XeOp __attribute__((ext_vector_type(4)));  // eight values of a matrix instruction's operand

constexpr int kXeWaves = kBlock / kWave;
constexpr int kXeChunk = 1024;  // bytes of an operand of one matrix instruction
constexpr int kXeMaxParts = 64;  // of a group whose rows are kept (a loss)
constexpr int kXeMaxDim = 512;
constexpr float kXeLog2e = 1.44269504088896340736f;
constexpr float kXeLn2 = 0.69314718055994530942f;
constexpr float kXeLeftOut = -1e30f;  // a bias of this or less leaves its class out, as -infinity does
constexpr float kXeStep = 8.0f;       // powers of two that a row's values may pass its running maximum by

enum { kXeLoss = 0, kXeLossAndRows = 1, kXeWeights = 2 };

// A tile's first kilobyte, in floats.  Classes: their biases.  Rows: -maximum (powers of two), factor, label, the label's value.
constexpr int kXeShift = 0, kXeFactor = 32, kXeLabel = 64, kXeOwn = 96;

// Sizes of a problem as the kernels see it: blocks of 32 columns, padded.  Beyond 256 columns in bf16, 320 in fp32, in two slices, each with half of O,
// which otherwise did not fit a wave's registers.  bf16 forms S for either.  In fp32 half of the columns of the kept rows is all that fits beside half of
// O too: two waves share them, each forms its half of S, and they add the halves up.  (8192 rows, 10 K classes, 512 columns, forward and backward: 2076
// us, 3140 with S formed for either and the kept rows' other half read from the L2 for each tile, 2293 by the library; 384 columns 1608, 1835 with S
// formed for either, 1800 by the library.)  (bf16 could have 384 columns whole, with one wave a SIMD instead of
// two: 8192 rows, 20 K classes, forward, 300 columns 340 us against 352 in slices, 370 columns 556 against 352.)
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
    s.slices = n > (s.parts == 3 ? 10 : 8) ? 2 : 1;
    const int blocks = n <= 8 ? n : n <= 10 && s.parts == 3 ? 10 : n <= 12 ? 12 : 16;
    s.blocks = blocks / s.slices;
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
    int* done;  // cleared: workgroups of xe_combine_kernel that have left their tile's loss
};

constexpr int kXeCols = 128;  // columns that a workgroup lays out, of 32 rows
constexpr int kXePitch = kXeCols + 4;

__device__ __forceinline__ XeOp xe_bf16(const float (&v)[8])
{
    Bf16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (__bf16)v[j];
    return __builtin_bit_cast(XeOp, o);
}

// Eight values as an operand of one matrix instruction, or as three
template <int PARTS>
__device__ __forceinline__ void xe_operands(const float (&v)[8], XeOp (&p)[PARTS])
{
    if constexpr (PARTS == 3) {
        uint32_t rest = 0;  // (bits below 2^-133: nothing beside a logit, and beside a gradient of x's own size)
        sp_split(v, p, rest);
    } else {
        p[0] = xe_bf16(v);
    }
}

template <int PARTS>
__device__ __forceinline__ void xe_put(const float (&v)[8], char* to)
{
    XeOp p[PARTS];
    xe_operands<PARTS>(v, p);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) *reinterpret_cast<XeOp*>(to + q * kXeChunk) = p[q];
}

template <typename T, int PARTS>
__global__ __launch_bounds__(kBlock) void xe_images_kernel(const XeImagesArgs g)
{
    __shared__ float tile[32 * kXePitch];
    __shared__ int live[32];  // rows that there are, and that have a label; classes that no bias leaves out: the others are taken as zeros
    const int64_t id = blockIdx.x;
    const bool classes = id >= g.first_tiles;
    const XeMatrix& m = g.m[classes ? 1 : 0];
    const int64_t t = classes ? id - g.first_tiles : id, row0 = 32 * t;
    const int col0 = kXeCols * (int)blockIdx.y, thread = (int)threadIdx.x;
    const T* src = static_cast<const T*>(m.src);
    if (id == 0 && blockIdx.y == 0 && thread == 0) *g.done = 0;
    float bias = -INFINITY;
    int label = -1;  // none
    if (thread < 32) {
        const int64_t row = row0 + thread;
        if (row < m.rows) {
            if (classes) {
                bias = m.bias != nullptr ? (float)static_cast<const T*>(m.bias)[row] : 0.0f;
                if (bias <= kXeLeftOut) bias = -INFINITY;
            } else {
                const int64_t y = g.label64 ? static_cast<const int64_t*>(m.labels)[row] : (int64_t) static_cast<const int32_t*>(m.labels)[row];
                if (y != g.ignore) label = y >= 0 && y < g.classes ? (int)y : -2;  // (-2: no such class)
            }
        }
        live[thread] = row < m.rows && (classes ? bias != -INFINITY : label != -1);
    }
    __syncthreads();
    if (m.col_stride == 1) {
        typedef T Vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
#pragma unroll
        for (int k = 0; k < 32 * kXeCols / 8 / kBlock; ++k) {
            const int at = thread + k * kBlock, r = at / (kXeCols / 8), c = at % (kXeCols / 8) * 8, left = g.dim - col0 - c;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.0f;
            if (live[r]) {
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
            tile[r * kXePitch + c] = live[r] && col0 + c < g.dim ? (float)src[(row0 + r) * m.row_stride + (col0 + c) * m.col_stride] : 0.0f;
        }
    }
    const int all_blocks = g.blocks * g.slices, steps = 2 * all_blocks;
    char* s_tile = m.s_image + t * kXeChunk * (1 + (int64_t)steps * PARTS);
    if (blockIdx.y == 0 && thread < 32) {
        if (classes) reinterpret_cast<float*>(s_tile)[thread] = bias;
        else reinterpret_cast<int*>(s_tile)[kXeLabel + thread] = label;
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
// How the groups' tiles are dealt out to workgroups.
struct XePlan {
    int groups;  // of four kept tiles (times slices), or of two, for the pairs of waves
    int slices;
    bool pairs;
    int tiles;   // passed, of each
    int per;     // tiles of a workgroup, of those that are shared
    int shared;  // > 0: that many workgroups to a group
    // shared = 0: each of `room` workgroups has whole groups, one in every round, of the first `whole` ones, all at the same tile at the same time (which
    // the XCDs' L2s are for), and then `per` tiles of the others', counted through without regard for the groups' ends
    int room, whole;

    int64_t workgroups() const { return shared > 0 ? (int64_t)groups * shared : room; }
    int64_t slots() const { return shared > 0 ? (int64_t)groups * shared : (int64_t)room + groups; }  // parts of groups at most
    // A group's first and last workgroup among those that share it, and the place of one's part
    __host__ __device__ int first(int group) const { return shared > 0 ? group * shared : group < whole ? 0 : (group - whole) * tiles / per; }
    __host__ __device__ int last(int group) const { return shared > 0 ? group * shared + shared - 1 : group < whole ? 0 : ((group - whole + 1) * tiles - 1) / per; }
    // Who has a tile's slice
    __host__ __device__ int group_of(int tile, int slice) const { return pairs ? tile / (kXeWaves / 2) : tile / kXeWaves * slices + slice; }
    __host__ __device__ int wave_of(int tile, int slice) const { return pairs ? tile % (kXeWaves / 2) * 2 + slice : tile % kXeWaves; }
    __host__ __device__ int slot(int workgroup, int group) const { return shared > 0 ? workgroup : group < whole ? group : group + workgroup; }
};

// Memory that all lanes have in common, its address in scalar registers: the compiler otherwise adds a lane's part to what the loops have in
// common and keeps the sums in registers.
template <typename T>
using XeGlobal = __attribute__((address_space(1))) T;
template <typename T>
__device__ __forceinline__ XeGlobal<T>* xe_uniform(T* p)
{
    XeGlobal<T>* q = (XeGlobal<T>*)p;
    asm("" : "+s"(q));
    return q;
}

// The loss's gradient for all rows, where it is the same for all: of a sum, or of a mean over the rows that have a label.
struct XeFactor {
    const float* d_loss;  // null: rows have one each, which is in their factors
    const float* count;   // or null
    __device__ __forceinline__ float value() const
    {
        if (d_loss == nullptr) return 1.0f;
        return count == nullptr ? *d_loss : *count > 0.0f ? *d_loss / *count : 0.0f;  // (no labels at all: no gradients)
    }
};

struct XeArgs {
    XePlan plan;
    const char* kept;      // S images
    const char* passed;
    const char* passed_p;  // P image
    int kept_tiles;
    float* stats;  // [slot][wave][row of 32]: maximum, others' sum, label's logit (powers of two), -  (weights: sum, -, -, -)
    float* part;   // [slot][wave][block][quarter][lane][4]
    XeFactor factor;      // weights: of all results
    // weights of groups that one workgroup has alone: straight to the result
    void* d_w;
    void* d_b;
    int64_t kept_rows;
    int dim;
};

// The value that the lane with the same kept row in the wave's other half has.
__device__ __forceinline__ float xe_other_half(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);  // (the lower lanes' values, the upper ones')
    return __uint_as_float(lane_id() < 32 ? r[1] : r[0]);
}

// A wave's part of a copy of CHUNKS kilobytes to LDS, past the registers.  (Through a buffer's descriptor: after a copy from a plain address, which
// might be LDS for all that the compiler knows, it waits for every read of LDS before it uses the first.)
template <int CHUNKS>
__device__ __forceinline__ void xe_stage(const char* src, char* dst)
{
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave)), lane = lane_id();
    const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(src), 0, CHUNKS * kXeChunk, 0x00027000);
#pragma unroll
    for (int c0 = 0; c0 < CHUNKS; c0 += kXeWaves) {
        const int c = c0 + wave;
        if (CHUNKS % kXeWaves == 0 || c < CHUNKS)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(dst + c * kXeChunk), 16, lane * 16, c * kXeChunk, 0, 0);
    }
}

__device__ __forceinline__ void xe_staged()
{
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies have arrived
    __syncthreads();
}

__device__ __forceinline__ XeOp xe_operand(const char* chunk) { return *reinterpret_cast<const XeOp*>(chunk + lane_id() * 16); }

__device__ __forceinline__ XeOp xe_operand(const XeGlobal<const char>* chunk) { return *reinterpret_cast<const XeGlobal<const XeOp>*>(chunk + lane_id() * 16); }

__device__ __forceinline__ XeF32x16 xe_mfma(const XeOp& a, const XeOp& b, const XeF32x16& c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0, 0, 0);
}

// N products of an operand from LDS each, in PARTS parts at neighbouring places: at(i) is the i-th one's place, use(i, parts) multiplies.  Operands are
// read a few products before they are used, and the compiler is kept from moving either: left to itself it reads two, waits for them and
// multiplies.
template <int N, int PARTS, typename At, typename Use>
__device__ __forceinline__ void xe_products(const At& at, const Use& use)
{
    constexpr int kMost = PARTS == 1 ? 4 : 2, kAhead = N < kMost ? N : kMost;
    XeOp a[kAhead][PARTS];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) a[i][p] = xe_operand(at(i) + p * kXeChunk);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        use(i, a[i % kAhead]);
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
            if (i + kAhead < N) a[i % kAhead][p] = xe_operand(at(i + kAhead) + p * kXeChunk);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// a b + c, in three parts: the small products first
__device__ __forceinline__ XeF32x16 xe_mfma(const XeOp (&a)[3], const XeOp (&b)[3], XeF32x16 c)
{
    constexpr int kA[6] = {2, 0, 1, 1, 0, 0}, kB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
    for (int q = 0; q < 6; ++q) c = xe_mfma(a[kA[q]], b[kB[q]], c);
    return c;
}
__device__ __forceinline__ XeF32x16 xe_mfma(const XeOp (&a)[1], const XeOp (&b)[1], const XeF32x16& c) { return xe_mfma(a[0], b[0], c); }

// Waves that a SIMD (and so workgroups that a CU) holds at once: the kept rows take 8 registers a block and part, O 16 a block, of 512.  (The loss
// alone in fp32, 7 blocks and more: LDS has room for one workgroup.)  WIDE: in two slices.
__host__ __device__ constexpr int xe_waves(int blocks, int parts, int use, bool wide)
{
    if (wide) return parts == 1 && (use == kXeLoss || blocks <= 6) ? 2 : 1;
    if (use == kXeLoss) return parts == 1 ? 4 : blocks <= 2 ? 4 : blocks <= 4 ? 3 : blocks <= 6 ? 2 : 1;
    return parts == 1 ? (blocks <= 2 ? 4 : blocks <= 3 ? 3 : 2) : blocks <= 1 ? 4 : blocks <= 2 ? 3 : blocks <= 4 ? 2 : 1;
}

// fp32 in two slices: neighbouring waves share their kept rows, each with the columns of its slice.
__host__ __device__ constexpr bool xe_pair(int parts, int use, bool wide) { return wide && parts == 3 && use != kXeLoss; }

template <int DB, int PARTS, int USE, bool WIDE>
struct XeWave {
    static constexpr int kSteps = WIDE ? 4 * DB : 2 * DB;
    static constexpr int kSChunks = 1 + kSteps * PARTS, kPChunks = 2 * DB * PARTS;

    static constexpr bool kPair = xe_pair(PARTS, USE, WIDE);
    static constexpr int kKept = kPair ? kSteps / 2 : kSteps;  // (a wave of a pair: its half of the columns)

    XeOp kept[kKept][PARTS];
    XeF32x16 o[USE == kXeLoss ? 1 : DB];
    float start;          // weights: the class's bias
    float top, sum, own;  // running maximum (a power of two), sum, the label's logit (a power of two)
    int label;            // weights: the class
    bool bias_sum;

    // What S^T of a tile starts from: the biases
    __device__ __forceinline__ XeF32x16 biases(const char* tile) const
    {
        XeF32x16 acc;
        if constexpr (USE == kXeWeights) {
            float bias = start;
            asm volatile("" : "+v"(bias));  // (else sixteen copies of it are kept in registers through all tiles)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] = bias;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const XeF4 b = of_rows(tile, 0, q);
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[4 * q + c] = b[c];
            }
        }
        return acc;
    }
    // acc and the products of the kept rows, from step FIRST on, with operands that lie one after another
    template <int FIRST>
    __device__ __forceinline__ XeF32x16 logits(const char* s, XeF32x16 acc) const
    {
        constexpr int kN = kPair ? DB : kKept;
        xe_products<kN, PARTS>([&](int k) { return s + k * PARTS * kXeChunk; }, [&](int k, const XeOp (&a)[PARTS]) { acc = xe_mfma(a, kept[FIRST + k], acc); });
        return acc;
    }
    // S^T of the staged tile
    __device__ __forceinline__ XeF32x16 logits(const char* s) const { return logits<0>(s + kXeChunk, biases(s)); }

    // Four values of the staged tile's rows that a lane's values 4 q .. 4 q + 3 of S^T belong to.
    static __device__ __forceinline__ XeF4 of_rows(const char* tile, int what, int q)
    {
        return *reinterpret_cast<const XeF4*>(reinterpret_cast<const float*>(tile) + what + 8 * q + 4 * (lane_id() / 32));
    }

    // S^T -> P^T, with the running maximum, sum and the label's logit.  v0: the tile's first class.
    __device__ __forceinline__ void shares(XeF32x16& s, int v0)
    {
        const int in_tile = label - v0;
        const bool here = label >= 0 && in_tile >= 0 && in_tile < 32;
        if (__any(here)) {
            const int at = here ? in_tile - 4 * (lane_id() / 32) : -1;  // (of the lane's values, if it has it)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (at == 8 * (i / 4) + i % 4) {
                    own = s[i] * kXeLog2e;
                    s[i] = -INFINITY;
                }
            }
        }
        float most = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) most = fmaxf(most, s[i]);
        most = fmaxf(most, xe_other_half(most)) * kXeLog2e;
        if (__any(most > top + kXeStep)) {
            const float now = fmaxf(top, most);
            const float scale = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= scale;
            if constexpr (USE == kXeLossAndRows) rescale(scale);
        }
        const float shift = top == -INFINITY ? 0.0f : -top;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], kXeLog2e, shift));
        add_up(s);
    }

    __device__ __forceinline__ void rescale(float scale)
    {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= scale;
    }

    __device__ __forceinline__ void add_up(const XeF32x16& p)
    {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = p[i] + p[i + 8];
        sum += (((t[0] + t[4]) + (t[1] + t[5])) + ((t[2] + t[6]) + (t[3] + t[7])));
    }

    // S^T -> the gradient of the logits, from the maxima, factors and labels of the tile's rows.  Returns whether a label is among them.
    __device__ __forceinline__ bool gradients(XeF32x16& s, const char* tile, int v0)
    {
        const int* l = reinterpret_cast<const int*>(tile);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const XeF4 shift = of_rows(tile, kXeShift, q), factor = of_rows(tile, kXeFactor, q);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                s[4 * q + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * q + j], kXeLog2e, shift[j])) * factor[j];
        }
        const int in_tile = l[kXeLabel + lane_id() % 32] - v0;
        const bool labels_here = __any(in_tile >= 0 && in_tile < 32);
        if (labels_here) {
            typedef int I4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const I4 labels = __builtin_bit_cast(I4, of_rows(tile, kXeLabel, q));
                const XeF4 values = of_rows(tile, kXeOwn, q);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * q + j] = labels[j] == label ? values[j] : s[4 * q + j];
            }
        }
        if (bias_sum) add_up(s);
        return labels_here;
    }

    // O^T += passed^T P^T.  both: bf16, P in two parts.
    __device__ __forceinline__ void product(const XeF32x16& s, const char* p, bool both)
    {
        XeOp w[2][PARTS];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = s[8 * h + j];
            xe_operands<PARTS>(v, w[h]);
        }
        if constexpr (PARTS == 1) {
            xe_products<2 * DB, 1>([&](int i) { return p + i * kXeChunk; }, [&](int i, const XeOp (&a)[1]) { o[i % DB] = xe_mfma(a, w[i / DB], o[i % DB]); });
            // A class's gradient is mostly its own rows' where there are many classes: those tiles take what rounding left of P too (the error
            // of dw against 64 bits, 1000 rows and 10 K classes: 2.4e-3 without, 1.7e-3 with, as its own rounding to bf16 makes).
            if (USE == kXeWeights && both) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[8];
                    const Bf16x8 high = __builtin_bit_cast(Bf16x8, w[h][0]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = s[8 * h + j] - (float)high[j];
                    w[h][0] = xe_bf16(v);
                }
                xe_products<2 * DB, 1>([&](int i) { return p + i * kXeChunk; }, [&](int i, const XeOp (&a)[1]) { o[i % DB] = xe_mfma(a, w[i / DB], o[i % DB]); });
            }
        } else {
            // Where O lies in the accumulator registers, the compiler moves it back and forth for instructions that add to it: it is added to in
            // fp32 instead, while the next block is multiplied (8192 rows, 20 K classes, forward and backward, added to so and by the matrix
            // instructions: 256 columns 1635 us and 1797, 200 columns 1428 and 1444; 128 columns 845 and 782, 64 columns 503 and 432).
            constexpr bool kOwn = DB > 4;
            XeF32x16 sum[2];
            xe_products<2 * DB, PARTS>([&](int i) { return p + (i % 2 * DB + i / 2) * PARTS * kXeChunk; }, [&](int i, const XeOp (&a)[PARTS]) {
                if constexpr (kOwn) {
                    XeF32x16& to = sum[i / 2 % 2];
                    to = xe_mfma(a, w[i % 2], i % 2 == 0 ? XeF32x16{} : to);
                    if (i >= 2 && i % 2 == 0) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) o[i / 2 - 1][c] += sum[(i / 2 - 1) % 2][c];
                    }
                } else {
                    o[i / 2] = xe_mfma(a, w[i % 2], o[i / 2]);
                }
            });
            if constexpr (kOwn) {
#pragma unroll
                for (int c = 0; c < 16; ++c) o[DB - 1][c] += sum[(DB - 1) % 2][c];
            }
        }
    }

    // Half of the steps of a pair's tile, of either slice, to one place: the first or the second half of each slice's operands of S, or of O
    static constexpr int kPiece = 2 * DB * PARTS * kXeChunk;
    static __device__ __forceinline__ void stage_piece(const char* tile, int half, char* to)
    {
        xe_stage<DB * PARTS>(tile + half * (kPiece / 2), to);
        xe_stage<DB * PARTS>(tile + kPiece + half * (kPiece / 2), to + kPiece / 2);
    }
    // One tile of a pair, whose S and P go through LDS in four such pieces, each in one of three places (arrays of their own: in one array, all reads wait
    // for the copies; 512 columns 2261 us for 2076).  At the start a and b have S, in the end b and c the next tile's; next: that, or null.
    __device__ __forceinline__ void pair_tile(char* a, char* b, char* c, char* header, const char* of_p, const char* next, int slice, int n0, int v0, bool active)
    {
        const int own = slice * (kPiece / 2), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
        stage_piece(of_p, 0, c);
        XeF32x16 p = {};
        if (active) {
            if (slice == 0) p = biases(header);
            p = logits<0>(a + own, p);
            p = logits<DB>(b + own, p);
        }
        __syncthreads();
        // the other wave's half of S is added (the same sum for both)
        XeF4* mine = reinterpret_cast<XeF4*>(a) + wave * 4 * kWave + lane_id();
        const XeF4* others = reinterpret_cast<const XeF4*>(a) + (wave ^ 1) * 4 * kWave + lane_id();
        if (active) {
#pragma unroll
            for (int q = 0; q < 4; ++q) mine[q * kWave] = XeF4{p[4 * q], p[4 * q + 1], p[4 * q + 2], p[4 * q + 3]};
        }
        __syncthreads();
        XeOp w[2][PARTS];
        if (active) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const XeF4 v = others[q * kWave];
#pragma unroll
                for (int j = 0; j < 4; ++j) p[4 * q + j] += v[j];
            }
            if constexpr (USE == kXeWeights) gradients(p, header, v0);
            else shares(p, n0);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = p[8 * h + j];
                xe_operands<PARTS>(v, w[h]);
            }
        }
        xe_staged();
        stage_piece(of_p, 1, a);
        if (next != nullptr) {
            xe_stage<1>(next, header);
            stage_piece(next + kXeChunk, 0, b);
        }
        if (active) half_product(w[0], c + own);
        xe_staged();
        if (next != nullptr) stage_piece(next + kXeChunk, 1, c);
        if (active) half_product(w[1], a + own);
        xe_staged();
    }

    // O^T += passed^T P^T of one half of a tile's passed rows
    __device__ __forceinline__ void half_product(const XeOp (&w)[PARTS], const char* p)
    {
        XeF32x16 sum[2];
        xe_products<DB, PARTS>([&](int i) { return p + i * PARTS * kXeChunk; }, [&](int i, const XeOp (&a)[PARTS]) {
            sum[i % 2] = xe_mfma(a, w, XeF32x16{});
            if (i == 0) return;
#pragma unroll
            for (int c = 0; c < 16; ++c) o[i - 1][c] += sum[(i - 1) % 2][c];
        });
#pragma unroll
        for (int c = 0; c < 16; ++c) o[DB - 1][c] += sum[(DB - 1) % 2][c];
    }

    // One tile: copies what comes next to `next` while it works on `s`
    __device__ __forceinline__ void first_half(const char* __restrict__ s, char* __restrict__ next, const char* src, XeF32x16& p, bool& both, int n0, int v0, bool active)
    {
        if constexpr (USE == kXeLoss) {
            if (src != nullptr) xe_stage<kSChunks>(src, next);
        } else {
            xe_stage<kPChunks>(src, next);
        }
        if (!active) return;
        p = logits(s);
        if constexpr (USE == kXeWeights) both = gradients(p, s, v0);
        else shares(p, n0);
    }
    // The same where LDS has room for two S tiles: the next one is on its way from the start of this one
    __device__ __forceinline__ void first_half_of_two(const char* __restrict__ s, char* __restrict__ next_p, char* __restrict__ next_s, const char* src_p, const char* src_s,
                                                      XeF32x16& p, bool& both, int n0, int v0, bool active)
    {
        xe_stage<kPChunks>(src_p, next_p);
        if (src_s != nullptr) xe_stage<kSChunks>(src_s, next_s);
        if (!active) return;
        p = logits(s);
        if constexpr (USE == kXeWeights) both = gradients(p, s, v0);
        else shares(p, n0);
    }
    // The same where LDS has room for two tiles of both: the next one is on its way all the while
    __device__ __forceinline__ void tile(const char* __restrict__ s, const char* __restrict__ p_tile, char* __restrict__ next_s, char* __restrict__ next_p, const char* src_s,
                                         const char* src_p, int n0, int v0, bool active)
    {
        if (src_s != nullptr) {
            xe_stage<kSChunks>(src_s, next_s);
            xe_stage<kPChunks>(src_p, next_p);
        }
        if (!active) return;
        XeF32x16 p = logits(s);
        bool both = false;
        if constexpr (USE == kXeWeights) both = gradients(p, s, v0);
        else shares(p, n0);
        product(p, p_tile, both);
    }
    __device__ __forceinline__ void second_half(const char* __restrict__ s, char* __restrict__ next, const char* src, const XeF32x16& p, bool both, bool active)
    {
        if (src != nullptr) xe_stage<kSChunks>(src, next);
        if (active) product(p, s, both);
    }
};

// Four neighbouring columns of a result's row, as far as it has them; as one where all rows have whole fours.
template <typename T>
__device__ __forceinline__ void xe_store4(T* row, int col, int dim, const XeF4& v)
{
    typedef T Vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (dim % 4 == 0) {
        if (col < dim) *reinterpret_cast<Vec*>(row + col) = Vec{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (col + c < dim) row[col + c] = (T)v[c];
    }
}
__device__ __forceinline__ void xe_store4(void* out, bool bf16, int64_t row, int col, int dim, const XeF4& v)
{
    if (bf16) xe_store4(static_cast<__bf16*>(out) + row * dim, col, dim, v);
    else xe_store4(static_cast<float*>(out) + row * dim, col, dim, v);
}

// What a lane has of a class's gradients, the class a group's alone.
template <typename T, int DB>
__device__ __forceinline__ void xe_store_weights(const XeArgs& g, const XeF32x16 (&o)[DB], int64_t row, int slice, float sum)
{
    if (row >= g.kept_rows) return;
    const float f = g.factor.value();
    int half = lane_id() / 32;
    asm volatile("" : "+v"(half));  // (else what the columns make of it is kept in registers through all tiles)
    if (g.d_b != nullptr && half == 0 && slice == 0) static_cast<T*>(g.d_b)[row] = (T)(sum * f);
    T* to = static_cast<T*>(g.d_w) + row * g.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            xe_store4(to, 32 * (slice * DB + d) + 8 * q + 4 * half, g.dim,
                      XeF4{o[d][4 * q] * f, o[d][4 * q + 1] * f, o[d][4 * q + 2] * f, o[d][4 * q + 3] * f});
}

template <int DB, int PARTS, int USE, bool WIDE>
__global__ __launch_bounds__(kBlock, xe_waves(DB, PARTS, USE, WIDE)) void xe_kernel(const XeArgs g)
{
    using Wave = XeWave<DB, PARTS, USE, WIDE>;
    // bf16 and 161 columns or more, the loss and its rows: two tiles of both in LDS, and one wait and barrier a tile.  (8192 rows, 40 K classes, forward, 256
    // columns 345 us so and 357 with one tile, 300 columns 688 and 703, 192 columns 282 and 286; 128 columns and fp32 no difference.  The weights'
    // gradient, which has a second product for some tiles, has no registers left for the one loop body: 955 us for 353.)
    constexpr bool kAll = USE == kXeLossAndRows && PARTS == 1 && DB >= 6 && !(WIDE && DB == 8);
    constexpr bool kPair = Wave::kPair;
    __shared__ __attribute__((aligned(16))) char s_buf[kPair ? Wave::kPiece : (kAll ? 2 : 1) * Wave::kSChunks * kXeChunk];
    // the loss alone: two tiles in turn, or one where LDS has no room for two
    constexpr bool kInTurn = USE == kXeLoss && 2 * Wave::kSChunks <= 156;
    __shared__ __attribute__((aligned(16))) char p_buf[(kPair ? 1 : USE != kXeLoss ? (kAll ? 2 : 1) * Wave::kPChunks : kInTurn ? Wave::kSChunks : 1) * kXeChunk];
    // In slices S is most of the work and O too little to hide the next S tile's copy behind.  (8192 x 512, 10 K classes, backward 399 us with
    // one S tile, 348 with two; two of P as well, 1250 us for 1147 of 40 K classes, forward.  Slices of 192 columns, two waves a SIMD, have no registers left for it.)
    constexpr bool kTwo = WIDE && DB == 8 && PARTS == 1 && USE != kXeLoss;
    __shared__ __attribute__((aligned(16))) char s_other[kPair ? Wave::kPiece : kTwo ? Wave::kSChunks * kXeChunk : 16], third[kPair ? Wave::kPiece : 16];
    constexpr int kSlices = WIDE && USE != kXeLoss && !kPair ? 2 : 1;
    constexpr int64_t kSBytes = (int64_t)Wave::kSChunks * kXeChunk, kPBytes = (int64_t)Wave::kPChunks * (WIDE ? 2 : 1) * kXeChunk;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const XePlan plan = g.plan;
    int workgroup = (int)blockIdx.x;
    if (plan.shared > 0) {
        // The workgroups of an XCD, every eighth one, take neighbouring places in an order by the part of the passed tiles, so that its L2 has to hold
        // few of those parts
        const int all = plan.groups * plan.shared, xcd = workgroup % 8, place = all / 8 * xcd + (xcd < all % 8 ? xcd : all % 8) + workgroup / 8;
        workgroup = place % plan.groups * plan.shared + place / plan.groups;
    }
    // this workgroup's groups: whole ones first, then parts
    int next = workgroup, whole = plan.shared > 0 ? 0 : plan.whole, t0 = 0, left = 0;
    for (bool parts = false;;) {
    int group;
    if (next < whole) {
        group = next;
        next += plan.room;
        left = plan.tiles;
    } else if (!parts) {
        parts = true;
        const int later = plan.shared > 0 ? 0 : workgroup * plan.per / plan.tiles;
        group = plan.shared > 0 ? workgroup / plan.shared : whole + later;
        t0 = plan.shared > 0 ? workgroup % plan.shared * plan.per : workgroup * plan.per - later * plan.tiles;
        left = plan.shared > 0 && plan.per > plan.tiles - t0 ? plan.tiles - t0 : plan.per;
        next = group + 1;
        whole = 0;
        if (group >= plan.groups) break;
    } else {
        if (left <= 0 || next >= plan.groups) break;
        group = next++;
        t0 = 0;
    }
    const int t1 = left < plan.tiles - t0 ? t0 + left : plan.tiles;
    left -= t1 - t0;
    const int slice = kPair ? wave % 2 : group % kSlices, tile = kPair ? group * (kXeWaves / 2) + wave / 2 : group / kSlices * kXeWaves + wave;
    const bool active = tile < g.kept_tiles;
    const XeGlobal<const char>* own = xe_uniform(g.kept + (active ? tile : g.kept_tiles - 1) * kSBytes);

    Wave w;
#pragma unroll
    for (int k = 0; k < Wave::kKept; ++k)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) w.kept[k][p] = xe_operand(own + kXeChunk + (((kPair ? slice * Wave::kKept : 0) + k) * PARTS + p) * kXeChunk);
#pragma unroll
    for (int d = 0; d < (USE == kXeLoss ? 1 : DB); ++d) w.o[d] = XeF32x16{};
    w.top = -INFINITY;
    w.sum = w.own = 0.0f;
    w.bias_sum = g.d_b != nullptr;
    if constexpr (USE == kXeWeights) {
        w.label = 32 * tile + lane % 32;
        w.start = reinterpret_cast<const XeGlobal<const float>*>(own)[lane % 32];
    } else {
        w.label = reinterpret_cast<const XeGlobal<const int>*>(own)[kXeLabel + lane % 32];
    }

    const int v0 = 32 * tile;
    XeF32x16 p = {};
    bool both = false;
    if constexpr (kPair) {
        xe_stage<1>(g.passed + t0 * kSBytes, p_buf);
        Wave::stage_piece(g.passed + t0 * kSBytes + kXeChunk, 0, s_buf);
        Wave::stage_piece(g.passed + t0 * kSBytes + kXeChunk, 1, s_other);
    } else {
        xe_stage<Wave::kSChunks>(g.passed + t0 * kSBytes, s_buf);
    }
    if constexpr (kAll) xe_stage<Wave::kPChunks>(g.passed_p + slice * (int64_t)Wave::kPChunks * kXeChunk + t0 * kPBytes, p_buf);
    xe_staged();
    if constexpr (kPair) {
        const auto step = [&](int t, char* a, char* b, char* c) {
            w.pair_tile(a, b, c, p_buf, g.passed_p + t * kPBytes, t + 1 < t1 ? g.passed + (t + 1) * kSBytes : nullptr, slice, 32 * t, v0, active);
        };
        for (int t = t0; t < t1; t += 3) {
            step(t, s_buf, s_other, third);
            if (t + 1 == t1) break;
            step(t + 1, s_other, third, s_buf);
            if (t + 2 == t1) break;
            step(t + 2, third, s_buf, s_other);
        }
    } else if constexpr (kAll) {
        const char* passed_p = g.passed_p + slice * (int64_t)Wave::kPChunks * kXeChunk;
        int at_s = 0, at_p = 0;
        for (int t = t0; t < t1; ++t) {
            const int to_s = Wave::kSChunks * kXeChunk - at_s, to_p = Wave::kPChunks * kXeChunk - at_p;
            const bool more = t + 1 < t1;
            w.tile(s_buf + at_s, p_buf + at_p, s_buf + to_s, p_buf + to_p, more ? g.passed + (t + 1) * kSBytes : nullptr, more ? passed_p + (t + 1) * kPBytes : nullptr,
                   32 * t, v0, active);
            xe_staged();
            at_s = to_s;
            at_p = to_p;
        }
    } else if constexpr (USE == kXeLoss && !kInTurn) {
        for (int t = t0; t < t1; ++t) {
            w.first_half(s_buf, p_buf, nullptr, p, both, 32 * t, v0, active);
            __syncthreads();
            if (t + 1 < t1) xe_stage<Wave::kSChunks>(g.passed + (t + 1) * kSBytes, s_buf);
            xe_staged();
        }
    } else if constexpr (USE == kXeLoss) {
        for (int t = t0; t < t1; t += 2) {
            w.first_half(s_buf, p_buf, t + 1 < t1 ? g.passed + (t + 1) * kSBytes : nullptr, p, both, 32 * t, v0, active);
            xe_staged();
            if (t + 1 == t1) break;
            w.first_half(p_buf, s_buf, t + 2 < t1 ? g.passed + (t + 2) * kSBytes : nullptr, p, both, 32 * (t + 1), v0, active);
            xe_staged();
        }
    } else if constexpr (kTwo) {
        const char* passed_p = g.passed_p + slice * (int64_t)Wave::kPChunks * kXeChunk;
        for (int t = t0; t < t1; t += 2) {
            w.first_half_of_two(s_buf, p_buf, s_other, passed_p + t * kPBytes, t + 1 < t1 ? g.passed + (t + 1) * kSBytes : nullptr, p, both, 32 * t, v0, active);
            xe_staged();
            if (active) w.product(p, p_buf, both);
            __syncthreads();
            if (t + 1 == t1) break;
            w.first_half_of_two(s_other, p_buf, s_buf, passed_p + (t + 1) * kPBytes, t + 2 < t1 ? g.passed + (t + 2) * kSBytes : nullptr, p, both, 32 * (t + 1), v0, active);
            xe_staged();
            if (active) w.product(p, p_buf, both);
            __syncthreads();
        }
    } else {
        const char* passed_p = g.passed_p + slice * (int64_t)Wave::kPChunks * kXeChunk;
        for (int t = t0; t < t1; ++t) {
            w.first_half(s_buf, p_buf, passed_p + t * kPBytes, p, both, 32 * t, v0, active);
            xe_staged();
            w.second_half(p_buf, s_buf, t + 1 < t1 ? g.passed + (t + 1) * kSBytes : nullptr, p, both, active);
            xe_staged();
        }
    }
    if (!active) continue;

    w.sum += xe_other_half(w.sum);
    w.own += xe_other_half(w.own);
    if constexpr (USE == kXeWeights) {
        if (t1 - t0 == plan.tiles) {
            xe_store_weights<typename std::conditional<PARTS == 1, __bf16, float>::type>(g, w.o, v0 + lane % 32, slice, w.sum);
            continue;
        }
    }
    const int64_t place = (int64_t)plan.slot(workgroup, group) * kXeWaves + wave;
    if (lane < 32) {  // (of either slice: they are cut in other places)
        const XeF4 v = USE == kXeWeights ? XeF4{w.sum, 0.0f, 0.0f, 0.0f} : XeF4{w.top, w.sum, w.own, 0.0f};
        *reinterpret_cast<XeGlobal<XeF4>*>(xe_uniform(g.stats + 4 * place * 32) + 4 * lane) = v;
    }
    if constexpr (USE != kXeLoss) {
        int at_lane = lane * 4;
        asm volatile("" : "+v"(at_lane));  // (as in xe_store_weights)
        XeGlobal<float>* to = xe_uniform(g.part + place * (DB * 4 * kWave * 4)) + at_lane;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<XeGlobal<XeF4>*>(to + (d * 4 + q) * kWave * 4) = XeF4{w.o[d][4 * q], w.o[d][4 * q + 1], w.o[d][4 * q + 2], w.o[d][4 * q + 3]};
    }
    }
}

// ---- what the parts of groups left, added up -----------------------------------------------------------------------
struct XeRow {  // of a row, for the backward pass
    float top, inverse, others;  // maximum (a power of two), 1 / sum, the other classes' share
    int label;
};

struct XeCombineArgs {
    XePlan plan;
    const float* stats;
    const float* part;
    char* rows;  // S image of the rows: their labels; what the weights' gradient needs of them goes there
    int64_t n_rows, s_bytes;
    int blocks, slices;
    const void* w;  // classes
    int64_t w_row, w_col;
    int dim, bf16;
    float* losses;     // a row each, or null
    float* tile_loss;  // [tile][2]: sum, count; or null
    int tiles, mean;
    int* done;
    float *loss, *count;
    XeRow* kept;  // or null
    int weights;  // whether their gradient is wanted
    float* d_x;   // [row][padded columns], up to its factor, or null
};

// The tiles' losses -> the loss, and the rows that have a label.  By the last workgroup that left one, in their order.
__device__ __forceinline__ void xe_total(const XeCombineArgs& g, double (&sums)[2][kXeWaves])
{
    double sum = 0.0, n = 0.0;
    for (int t = (int)threadIdx.x; t < g.tiles; t += kBlock) {
        sum += (double)__hip_atomic_load(g.tile_loss + 2 * t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        n += (double)__hip_atomic_load(g.tile_loss + 2 * t + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int d = kWave / 2; d >= 1; d >>= 1) {
        sum += __shfl_xor(sum, d, kWave);
        n += __shfl_xor(n, d, kWave);
    }
    if (lane_id() == 0) {
        sums[0][threadIdx.x / kWave] = sum;
        sums[1][threadIdx.x / kWave] = n;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
#pragma unroll
    for (int k = 1; k < kXeWaves; ++k) {
        sum += sums[0][k];
        n += sums[1][k];
    }
    *g.loss = (float)(g.mean ? sum / n : sum);  // (no labels at all: not a number, as the mean of nothing is)
    *g.count = (float)n;
}

// One workgroup a tile of 32 rows and block of 32 columns.  Each forms the rows' sums from their parts (a row eight threads), the first of
// a tile's keeps them; then a wave takes eight columns.  What it needs from memory is asked for at once, at the start: the time of such a
// launch is that of a few reads one after another.
__global__ __launch_bounds__(kBlock) void xe_combine_kernel(const XeCombineArgs g)
{
    constexpr int kEach = kBlock / 32, kFirst = 4;
    __shared__ float scale[kXeMaxParts * 32];
    __shared__ float top_of[kEach][32], own_of[kEach][32], rest_of[kEach][32];
    __shared__ double totals[2][kXeWaves];
    __shared__ int last;
    const int tile = (int)blockIdx.x, block = (int)blockIdx.y, group = g.plan.group_of(tile, block / g.blocks);
    const int64_t row0 = 32LL * tile;
    const int thread = (int)threadIdx.x, wave = g.plan.wave_of(tile, block / g.blocks), i = thread % 32, each = thread / 32, lane = thread % kWave;
    const int b0 = g.plan.first(group), parts = g.plan.last(group) - b0 + 1;
    const int64_t place = (int64_t)g.plan.slot(b0, group) * kXeWaves + wave, step = (int64_t)kXeWaves * g.blocks * 4 * kWave;
    const XeF4* s = reinterpret_cast<const XeF4*>(g.stats) + place * 32 + i;
    const XeF4* p = reinterpret_cast<const XeF4*>(g.part) + (place * g.blocks + block % g.blocks) * 4 * kWave + thread;
    char* own_tile = g.rows + tile * g.s_bytes;
    const bool there = row0 + i < g.n_rows, with_x = g.d_x != nullptr;
    const int col = 32 * block + thread / kWave * 8 + lane / 32 * 4;
    XeF4 mine = {-INFINITY, 0.0f, 0.0f, 0.0f}, first[kFirst];
    if (each < parts) mine = s[each * kXeWaves * 32];
    const int label = reinterpret_cast<const int*>(own_tile)[kXeLabel + i];
    if (with_x) {
#pragma unroll
        for (int k = 0; k < kFirst; ++k) first[k] = p[(k < parts ? k : 0) * step];
    }
    XeF4 w = {};
    if (with_x && label >= 0) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (col + c >= g.dim) continue;
            const int64_t from = label * g.w_row + (col + c) * g.w_col;
            w[c] = g.bf16 ? (float)static_cast<const __bf16*>(g.w)[from] : static_cast<const float*>(g.w)[from];
        }
    }
    float top = mine[0], own = mine[2];
    for (int k = each + kEach; k < parts; k += kEach) {
        const XeF4 v = s[k * kXeWaves * 32];
        top = fmaxf(top, v[0]);
        own += v[2];
    }
    top_of[each][i] = top;
    own_of[each][i] = own;
    __syncthreads();
    own = 0.0f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        top = fmaxf(top, top_of[k][i]);
        own += own_of[k][i];
    }
    if (label >= 0) top = fmaxf(top, own);
    float rest = 0.0f;
    for (int k = each; k < parts; k += kEach) {
        const XeF4 v = k == each ? mine : s[k * kXeWaves * 32];
        const float f = v[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v[0] - top);
        rest += v[0] == -INFINITY ? v[1] : v[1] * f;  // (what is not a number stays it)
        scale[k * 32 + i] = f;
    }
    rest_of[each][i] = rest;
    __syncthreads();
    rest = 0.0f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) rest += rest_of[k][i];
    const float own_part = label >= 0 ? __builtin_amdgcn_exp2f(own - top) : 0.0f;
    const float total = rest + own_part, inverse = 1.0f / total, others = label == -2 ? NAN : rest * inverse;
    if (with_x && there) {
        XeF4 sum = {};
#pragma unroll
        for (int k = 0; k < kFirst; ++k) {
            const float f = k < parts ? scale[k * 32 + i] : 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += k < parts ? first[k][c] * f : 0.0f;
        }
#pragma unroll 4
        for (int k = kFirst; k < parts; ++k) {
            const XeF4 v = p[k * step];
            const float f = scale[k * 32 + i];
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += v[c] * f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] = label >= 0 || label == -2 ? sum[c] * inverse - others * w[c] : 0.0f;
        *reinterpret_cast<XeF4*>(g.d_x + (row0 + i) * (32 * g.blocks * g.slices) + col) = sum;
    }
    if (block != 0) return;  // (the tile's first workgroup alone keeps what is the rows')
    if (thread < kWave) {
        float loss = top - own < 64.0f ? log1pf(rest / own_part) : kXeLn2 * (top - own) + logf(total);
        if (label == -2) loss = NAN;
        if (label == -1) loss = 0.0f;
        if (thread < 32) {
            if (there && g.losses != nullptr) g.losses[row0 + i] = loss;
            if (there && g.kept != nullptr) g.kept[row0 + i] = XeRow{top, inverse, others, label};
            if (g.weights) {  // (rows without a label and past the end: no share)
                float* c = reinterpret_cast<float*>(own_tile);
                c[kXeShift + i] = label == -1 ? -INFINITY : label == -2 ? NAN : -top;
                c[kXeFactor + i] = label == -1 ? 0.0f : inverse;
                c[kXeOwn + i] = -others;
            }
        }
        float sum = there ? loss : 0.0f, count = there && label != -1 ? 1.0f : 0.0f;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) {
            sum += __shfl_xor(sum, d, kWave);
            count += __shfl_xor(count, d, kWave);
        }
        if (thread == 0 && g.tile_loss != nullptr) {
            __hip_atomic_store(g.tile_loss + 2 * tile, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(g.tile_loss + 2 * tile + 1, count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            // The two are where all of the chip sees them once their stores are counted as done; a release would write the L2's other contents back
            // too, for each tile (8192 rows: 8 us of 19).
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            last = __hip_atomic_fetch_add(g.done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == g.tiles - 1;
        }
    }
    if (g.tile_loss == nullptr) return;
    __syncthreads();
    if (last) xe_total(g, totals);
}

// Reductions that leave a loss for each row: the rows' factors, of the losses' gradients.
__global__ __launch_bounds__(kBlock) void xe_factors_kernel(const XeRow* __restrict__ kept, const float* __restrict__ d_loss, int64_t n_rows, char* __restrict__ rows,
                                                            int64_t s_bytes)
{
    const int64_t row = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (row >= n_rows) return;
    const XeRow r = kept[row];
    float* c = reinterpret_cast<float*>(rows + row / 32 * s_bytes) + row % 32;
    const float f = d_loss[row];
    c[kXeFactor] = r.label == -1 ? 0.0f : f * r.inverse;
    c[kXeOwn] = -f * r.others;
}

struct XeFinishArgs {
    // dx (null: not wanted), 32 rows and 32 columns a workgroup, the first dx_groups of them
    const XeRow* kept;
    const float* d_x;
    const float* d_loss;  // of a row each, or null
    XeFactor factor;
    int64_t n_rows;
    int cols, dim, bf16;
    void* out;
    int dx_groups;
    // the weights' gradient from its parts
    XePlan plan;
    const float* stats;
    const float* part;
    int64_t n_classes;
    int blocks, slices, groups_per_tile;
    void* d_w;
    void* d_b;  // or null
};

__device__ __forceinline__ void xe_finish_rows(const XeFinishArgs& g)
{
    const int col_groups = (g.dim + 31) / 32, thread = (int)threadIdx.x;
    const int64_t row = 32LL * ((int)blockIdx.x / col_groups) + thread / 8;
    const int col = (int)blockIdx.x % col_groups * 32 + thread % 8 * 4;
    if (row >= g.n_rows || col >= g.dim) return;
    XeF4 v = *reinterpret_cast<const XeF4*>(g.d_x + row * g.cols + col);
    const int label = g.kept[row].label;
    const float f = g.d_loss != nullptr ? g.d_loss[row] : g.factor.value();
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = label != -1 ? v[c] * f : 0.0f;
    xe_store4(g.out, g.bf16 != 0, row, col, g.dim, v);
}

// What is left to do for the gradients: dx from what the forward pass made of it, and the weights' gradient from the parts of shared groups.  A
// wave takes 32 classes and eight columns; where there are many parts (TOGETHER), a workgroup's four share them.
template <bool TOGETHER>
__global__ __launch_bounds__(kBlock) void xe_finish_kernel(const XeFinishArgs g)
{
    __shared__ XeF4 sums[TOGETHER ? kXeWaves : 1][kWave];
    __shared__ float biases[TOGETHER ? kXeWaves : 1][32];
    const int id = (int)blockIdx.x - g.dx_groups;
    if (id < 0) return xe_finish_rows(g);
    const int tile = id / g.groups_per_tile, in_tile = id % g.groups_per_tile;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave)), lane = lane_id();
    const int chunk = TOGETHER ? in_tile : in_tile * kXeWaves + wave, slice = chunk / (4 * g.blocks);
    const int group = g.plan.group_of(tile, slice), b0 = g.plan.first(group), parts = g.plan.last(group) - b0 + 1;
    if (parts == 1) return;  // (stored as it was formed)
    const int64_t place = (int64_t)g.plan.slot(b0, group) * kXeWaves + g.plan.wave_of(tile, slice);
    const int each = TOGETHER ? (parts + kXeWaves - 1) / kXeWaves : parts, k0 = TOGETHER ? wave * each : 0, k1 = k0 + each < parts ? k0 + each : parts;
    const int64_t step = (int64_t)kXeWaves * g.blocks * 4 * kWave;
    const XeF4* p = reinterpret_cast<const XeF4*>(g.part) + place * (g.blocks * 4 * kWave) + chunk % (4 * g.blocks) * kWave + lane;
    const bool with_bias = g.d_b != nullptr && chunk == 0;
    XeF4 sum = {};
    float bias = 0.0f;
    if (with_bias) {
#pragma unroll 8
        for (int k = k0; k < k1; ++k) bias += g.stats[4 * ((place + (int64_t)k * kXeWaves) * 32 + lane % 32)];
    }
    constexpr int kBatch = TOGETHER ? 8 : 4;  // parts that are asked for at once
    for (int k = k0; k < k1; k += kBatch) {
        XeF4 v[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) v[j] = p[(k + j < k1 ? k + j : k) * step];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += k + j < k1 ? v[j][c] : 0.0f;
    }
    if constexpr (TOGETHER) {
        sums[wave][lane] = sum;
        if (lane < 32) biases[wave][lane] = bias;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int k = 1; k < kXeWaves; ++k) {
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += sums[k][lane][c];
            bias += biases[k][lane % 32];
        }
    }
    const int64_t row = 32LL * tile + lane % 32;
    if (row >= g.n_classes) return;
    const float f = g.factor.value();
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[c] *= f;
    xe_store4(g.d_w, g.bf16 != 0, row, 8 * chunk + lane / 32 * 4, g.dim, sum);
    if (with_bias && lane < 32) {
        if (g.bf16) static_cast<__bf16*>(g.d_b)[row] = (__bf16)(bias * f);
        else static_cast<float*>(g.d_b)[row] = bias * f;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------
inline XePlan xe_plan(const XeShape& s, int use, int kept_tiles, int passed_tiles)
{
    XePlan p;
    p.slices = use == kXeLoss ? 1 : s.slices;
    p.pairs = xe_pair(s.parts, use, s.slices == 2);
    p.groups = p.pairs ? (int)ceil_div(kept_tiles, kXeWaves / 2) : (int)ceil_div(kept_tiles, kXeWaves) * p.slices;
    p.tiles = passed_tiles;
    const int room = 256 * xe_waves(s.blocks, s.parts, use, s.slices == 2);
    // at least: so that a part's kept rows and results are little beside its tiles, and for a loss so many parts that the combining kernel holds their
    // sums in LDS.  (100 rows, 500 K classes, bf16: 410 us with 62 parts, 1230 with 16.  Weights, 100 K rows, 47 classes, bf16: backward 42 us with 512
    // parts, 53 with 128, 135 with 32, and 69 with 1024, which the kernel's first tile and last stores are much of.)
    int least = (int)ceil_div(passed_tiles, use == kXeWeights ? 512 : kXeMaxParts - 2);
    // Two tiles, unless all of them are few beside the chip.  (1000 rows x 256, 64 classes, forward and backward with one and two: bf16 31 us and 34, fp32 39 and
    // 47; 172 classes 37 and 36, 47 and 51.  8192 rows, bf16, 64 classes 51 and 50, 172 classes 69 and 57.)
    const bool few = (int64_t)p.groups * passed_tiles < room / 4;
    if (least < 2 && !few) least = 2;
    if (least > passed_tiles) least = passed_tiles;
    p.shared = p.groups < room ? room / p.groups : 1;
    p.per = (int)ceil_div(passed_tiles, p.shared);
    if (p.per < least) p.per = least;
    // The weights' gradient of a few tiles and many classes in bf16: parts would cost more to write and add up than they save.  (190 rows, 256 columns,
    // backward, whole and in parts: bf16, 4 K classes 19 us and 20, 16 K 19 and 25, 32 K 23 and 37; fp32, 8 K classes 37 and 24, 16 K 40 and 38, 32 K 48 and 46.)
    if (use == kXeWeights && passed_tiles <= 6 && s.parts == 1 && p.groups > 48) p.per = passed_tiles;
    p.shared = (int)ceil_div(passed_tiles, p.per);
    p.room = room;
    p.whole = 0;
    // Where that leaves an eighth of the chip idle, in the only round or the last of a few: no regard for the groups' ends.  (40 K rows x 256, 20 K
    // classes, bf16: forward 877 us so, 977 in whole groups; 100 K x 128, 10 K classes: 618 and 732.)
    const int64_t full = (int64_t)p.groups * p.shared, rounds = ceil_div(full, room);
    if (p.per > least && p.per > 6 && rounds <= 8 && full * 8 < rounds * room * 7 && (p.groups % room + 1LL) * passed_tiles < 1LL << 31) {
        p.whole = p.groups / room * room;
        p.per = (int)ceil_div((int64_t)(p.groups - p.whole) * passed_tiles, room);
        if (p.per < least) p.per = least;
        p.shared = 0;
    }
    return p;
}

struct XeProblem {
    int64_t n, classes;
    int row_tiles, class_tiles;
    int dim, dtype;
    XeShape shape;
};

inline bool xe_problem(int64_t n, int64_t classes, int dim, int dtype, XeProblem* p)
{
    if (n < 1 || n >= 1LL << 29 || classes < 1 || classes >= 1LL << 29 || dim < 1 || dim > kXeMaxDim || (dtype != FGL_F32 && dtype != FGL_BF16)) return false;
    p->n = n;
    p->classes = classes;
    p->dim = dim;
    p->dtype = dtype;
    p->row_tiles = (int)ceil_div(n, 32);
    p->class_tiles = (int)ceil_div(classes, 32);
    if (p->row_tiles + (int64_t)p->class_tiles >= 1 << 24 || p->row_tiles * ceil_div(dim, 32) >= 1 << 23) return false;  // (launches have fewer than 2^32 threads)
    p->shape = xe_shape(dim, dtype);
    return true;
}

// What a forward pass leaves for the backward one, and its scratch.
struct XeState {
    char *rows_s, *rows_p, *classes_s;  // (weights' gradient)
    XeRow* kept;
    float* d_x;
    float* count;
    int* done;
    size_t bytes;
};

inline XeState xe_state(const XeProblem& p, int want, void* base)
{
    Carver c(base);
    XeState s = {};
    s.count = c.take<float>(2);
    s.done = reinterpret_cast<int*>(s.count + 1);
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
    const XePlan plan = xe_plan(p.shape, use, p.row_tiles, p.class_tiles);
    Carver c(base);
    XeScratch s = {};
    if (!(want & FGL_XENT_WEIGHTS)) {
        s.rows_s = c.take<char>((size_t)(p.row_tiles * p.shape.s_bytes()));
        s.classes_s = c.take<char>((size_t)(p.class_tiles * p.shape.s_bytes()));
    }
    if (use == kXeLossAndRows) {
        s.classes_p = c.take<char>((size_t)(p.class_tiles * p.shape.p_bytes()));
        s.part = c.take<float>((size_t)plan.slots() * kXeWaves * 32 * 32 * p.shape.blocks);
    }
    s.stats = c.take<float>((size_t)plan.slots() * kXeWaves * 32 * 4);
    s.tile_loss = c.take<float>((size_t)p.row_tiles * 2);
    s.bytes = c.used();
    return s;
}

inline XeScratch xe_backward_scratch(const XeProblem& p, int want, void* base)
{
    Carver c(base);
    XeScratch s = {};
    if (want & FGL_XENT_WEIGHTS) {
        const XePlan plan = xe_plan(p.shape, kXeWeights, p.class_tiles, p.row_tiles);
        if (plan.shared != 1) {
            s.part = c.take<float>((size_t)plan.slots() * kXeWaves * 32 * 32 * p.shape.blocks);
            s.stats = c.take<float>((size_t)plan.slots() * kXeWaves * 32 * 4);
        }
    }
    s.bytes = c.used();
    return s;
}

template <int PARTS, int USE>
void launch_xe_parts(const XeShape& s, const XeArgs& g, unsigned workgroups, hipStream_t stream)
{
    const dim3 grid(workgroups), block(kBlock);
    if (s.slices == 2) {
        if (s.blocks == 6) hipLaunchKernelGGL((xe_kernel<6, PARTS, USE, true>), grid, block, 0, stream, g);
        else hipLaunchKernelGGL((xe_kernel<8, PARTS, USE, true>), grid, block, 0, stream, g);
        return;
    }
    if constexpr (PARTS == 3) {
        if (s.blocks == 10) {
            hipLaunchKernelGGL((xe_kernel<10, PARTS, USE, false>), grid, block, 0, stream, g);
            return;
        }
    }
    switch (s.blocks) {
    case 1: hipLaunchKernelGGL((xe_kernel<1, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 2: hipLaunchKernelGGL((xe_kernel<2, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 3: hipLaunchKernelGGL((xe_kernel<3, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 4: hipLaunchKernelGGL((xe_kernel<4, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 5: hipLaunchKernelGGL((xe_kernel<5, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 6: hipLaunchKernelGGL((xe_kernel<6, PARTS, USE, false>), grid, block, 0, stream, g); break;
    case 7: hipLaunchKernelGGL((xe_kernel<7, PARTS, USE, false>), grid, block, 0, stream, g); break;
    default: hipLaunchKernelGGL((xe_kernel<8, PARTS, USE, false>), grid, block, 0, stream, g); break;
    }
}

template <int USE>
void launch_xe(const XeShape& s, XeArgs& g, int passed_tiles, hipStream_t stream)
{
    g.plan = xe_plan(s, USE, g.kept_tiles, passed_tiles);
    if (s.parts == 3) launch_xe_parts<3, USE>(s, g, (unsigned)g.plan.workgroups(), stream);
    else launch_xe_parts<1, USE>(s, g, (unsigned)g.plan.workgroups(), stream);
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
    const dim3 grid((unsigned)(p.row_tiles + p.class_tiles), (unsigned)ceil_div(s.cols(), kXeCols)), block(kBlock);
    im.done = st.done;
    if (dtype == FGL_F32) hipLaunchKernelGGL((xe_images_kernel<float, 3>), grid, block, 0, to, im);
    else hipLaunchKernelGGL((xe_images_kernel<__bf16, 1>), grid, block, 0, to, im);
    FGL_CHECK_LAUNCH("xe_images_kernel");

    XeArgs g = {};
    g.kept = im.m[0].s_image;
    g.passed = im.m[1].s_image;
    g.passed_p = ws.classes_p;
    g.kept_tiles = p.row_tiles;
    g.stats = ws.stats;
    g.part = ws.part;
    if (want & FGL_XENT_ROWS) launch_xe<kXeLossAndRows>(s, g, p.class_tiles, to);
    else launch_xe<kXeLoss>(s, g, p.class_tiles, to);
    FGL_CHECK_LAUNCH("xe_kernel");

    XeCombineArgs c = {};
    c.plan = g.plan;
    c.stats = ws.stats;
    c.part = ws.part;
    c.rows = im.m[0].s_image;
    c.n_rows = n_rows;
    c.s_bytes = s.s_bytes();
    c.blocks = s.blocks;
    c.slices = want & FGL_XENT_ROWS ? s.slices : 1;
    c.w = d_w;
    c.w_row = w_row_stride;
    c.w_col = w_col_stride;
    c.dim = dim;
    c.bf16 = dtype == FGL_BF16;
    c.losses = reduction == FGL_REDUCE_NONE ? d_loss : nullptr;
    c.tile_loss = reduction == FGL_REDUCE_NONE ? nullptr : ws.tile_loss;
    c.tiles = p.row_tiles;
    c.mean = reduction == FGL_REDUCE_MEAN;
    c.done = st.done;
    c.loss = d_loss;
    c.count = st.count;
    c.kept = st.kept;
    c.weights = (want & FGL_XENT_WEIGHTS) != 0;
    c.d_x = st.d_x;
    hipLaunchKernelGGL(xe_combine_kernel, dim3((unsigned)p.row_tiles, want & FGL_XENT_ROWS ? (unsigned)(s.blocks * s.slices) : 1u), block, 0, to, c);
    FGL_CHECK_LAUNCH("xe_combine_kernel");
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
    FGL_REQUIRE(d_loss_grad && d_state && (d_dx == nullptr || (want & FGL_XENT_ROWS)) && ((d_dw == nullptr && d_db == nullptr) || (want & FGL_XENT_WEIGHTS)) &&
                    (d_db == nullptr || d_dw != nullptr),
                "linear_cross_entropy_backward: null pointer, or a gradient that the forward pass was not told of");
    const XeState st = xe_state(p, want, d_state);
    const XeScratch ws = xe_backward_scratch(p, want, d_ws);
    if (state_bytes < st.bytes || ws_bytes < ws.bytes || (d_ws == nullptr && ws.bytes > 0) || ((uintptr_t)d_state | (uintptr_t)d_ws) % 256 != 0) {
        set_error("linear_cross_entropy_backward: needs %zu bytes of state and %zu of workspace on 256-byte boundaries, got %zu and %zu", st.bytes, ws.bytes, state_bytes, ws_bytes);
        return FGL_ERR_WORKSPACE;
    }
    const XeShape& s = p.shape;
    const hipStream_t to = as_stream(stream);
    const dim3 block(kBlock);
    const XeFactor factor = {reduction == FGL_REDUCE_NONE ? nullptr : d_loss_grad, reduction == FGL_REDUCE_MEAN ? st.count : nullptr};
    XeArgs g = {};
    if (d_dw != nullptr) {
        if (reduction == FGL_REDUCE_NONE) {
            hipLaunchKernelGGL(xe_factors_kernel, dim3((unsigned)ceil_div(n_rows, kBlock)), block, 0, to, st.kept, d_loss_grad, n_rows, st.rows_s, s.s_bytes());
            FGL_CHECK_LAUNCH("xe_factors_kernel");
        }
        g.kept = st.classes_s;
        g.passed = st.rows_s;
        g.passed_p = st.rows_p;
        g.kept_tiles = p.class_tiles;
        g.stats = ws.stats;
        g.part = ws.part;
        g.factor = factor;
        g.d_w = d_dw;
        g.d_b = d_db;
        g.kept_rows = n_classes;
        g.dim = dim;
        launch_xe<kXeWeights>(s, g, p.row_tiles, to);
        FGL_CHECK_LAUNCH("xe_kernel");
    }
    const bool parts = d_dw != nullptr && g.plan.shared != 1;
    if (d_dx == nullptr && !parts) return FGL_OK;
    // (8192 x 256, 47 classes, fp32, 128 parts: backward 20 us with four waves on them, 28 with one; with eight parts there is no difference)
    const bool together = parts && g.plan.shared > 8;
    XeFinishArgs f = {};
    f.kept = st.kept;
    f.d_x = st.d_x;
    f.d_loss = reduction == FGL_REDUCE_NONE ? d_loss_grad : nullptr;
    f.factor = factor;
    f.n_rows = n_rows;
    f.cols = s.cols();
    f.dim = dim;
    f.bf16 = dtype == FGL_BF16;
    f.out = d_dx;
    const int64_t dx_groups = d_dx != nullptr ? (int64_t)p.row_tiles * ceil_div(dim, 32) : 0;
    f.plan = g.plan;
    f.stats = ws.stats;
    f.part = ws.part;
    f.n_classes = n_classes;
    f.blocks = s.blocks;
    f.slices = s.slices;
    f.groups_per_tile = (together ? 4 : 1) * s.blocks * s.slices;
    f.d_w = d_dw;
    f.d_b = d_db;
    const int64_t groups = dx_groups + (parts ? (int64_t)p.class_tiles * f.groups_per_tile : 0);
    f.dx_groups = (int)dx_groups;
    if (together) hipLaunchKernelGGL(xe_finish_kernel<true>, dim3((unsigned)groups), block, 0, to, f);
    else hipLaunchKernelGGL(xe_finish_kernel<false>, dim3((unsigned)groups), block, 0, to, f);
    FGL_CHECK_LAUNCH("xe_finish_kernel");
    return FGL_OK;
}
