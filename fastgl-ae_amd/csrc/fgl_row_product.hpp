// What the kernels of a dense layer's product over rows share: operands, and how a lane's columns of a row are stored.
#pragma once

#include "fgl_activation.hpp"
#include "fgl_common.hpp"

namespace fgl {

struct RowProductSide {
    const void* a;
    const void* b;
    int64_t lda, ldb;
    int k;  // 0: no such pair
};
// What follows a product: C = act(A B + bias) + residual, and what act's derivative will be formed from, the sums themselves or a bit for each
struct RowProductEpilogue {
    int act;               // kActNone ..
    const void* residual;  // (may be null) of C's sizes
    int64_t ldr;
    void* z;               // (may be null) A B + bias in C's type
    int64_t ldz;
    uint32_t* mask;        // (may be null) relu: bit c % 32 of word c / 32 of a row
    int64_t mask_ld;       // words a row
};
struct RowProductArgs {
    RowProductSide side[2];  // C = A0 B0 + A1 B1
    const void* bias;
    void* c;
    int64_t ldc, m;
    int n;
    int tiles_n;          // tiles of C along n
    int64_t row_blocks;   // workgroups along m
    int vec_log;          // (split products) log2 of the neighbouring columns a lane stores
    RowProductEpilogue then;  // (kRpThen)
};

__device__ __forceinline__ uint32_t rp_bf16_bits(float v) { return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v); }

// V neighbouring values as they lie in memory, and one of them
template <typename T, int V>
struct RpHeld {
    static constexpr int kWords = sizeof(T) == 4 ? V : (V + 1) / 2;
    typedef uint32_t Vec __attribute__((ext_vector_type(kWords), aligned(4)));
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* p)
    {
        if constexpr (sizeof(T) == 2 && V == 1) {
            w[0] = *p;
        } else {
            const Vec v = *reinterpret_cast<const Vec*>(p);
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = v[i];
        }
    }
    __device__ __forceinline__ float at(int t) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[t]);
        else return __uint_as_float(t & 1 ? w[t / 2] & 0xFFFF0000u : w[t / 2] << 16);
    }
};

// v += what p holds
template <typename T, int VB>
__device__ __forceinline__ void rp_add(const T* p, float (&v)[VB])
{
    if constexpr (sizeof(T) == 4) {
        typedef float Vec __attribute__((ext_vector_type(VB), aligned(4)));
        const Vec o = *reinterpret_cast<const Vec*>(p);
#pragma unroll
        for (int t = 0; t < VB; ++t) v[t] += o[t];
    } else if constexpr (VB == 1) {
        v[0] += __uint_as_float((uint32_t)*p << 16);
    } else {
        typedef uint32_t Vec __attribute__((ext_vector_type(VB / 2), aligned(4)));
        const Vec o = *reinterpret_cast<const Vec*>(p);
#pragma unroll
        for (int t = 0; t < VB; ++t) v[t] += __uint_as_float(t & 1 ? o[t / 2] & 0xFFFF0000u : o[t / 2] << 16);
    }
}

template <typename T, int VB>
__device__ __forceinline__ void rp_store(T* p, const float (&v)[VB])
{
    if constexpr (sizeof(T) == 4) {
        typedef float Vec __attribute__((ext_vector_type(VB), aligned(4)));
        Vec o;
#pragma unroll
        for (int t = 0; t < VB; ++t) o[t] = v[t];
        *reinterpret_cast<Vec*>(p) = o;
    } else if constexpr (VB == 1) {
        *reinterpret_cast<__bf16*>(p) = (__bf16)v[0];
    } else {
        typedef __bf16 Vec __attribute__((ext_vector_type(VB), aligned(4)));
        Vec o;
#pragma unroll
        for (int t = 0; t < VB; ++t) o[t] = (__bf16)v[t];
        *reinterpret_cast<Vec*>(p) = o;
    }
}

// FORM: one product (kRpOne), two of them and their sum (kRpSum: a layer's own rows with one weight and its gathered rows with another, in one
// pass over C where the products and their sum were five), or a product added to what C holds (kRpAdd).  In bf16 a product is rounded to
// bf16 before it is added to another or to C, as it would be if it were stored in between.
// kRpThen: one product and its epilogue.
constexpr int kRpOne = 0, kRpSum = 1, kRpAdd = 2, kRpThen = 3;

// The epilogue of 16 rows of a lane, of V neighbouring columns each from `col` on; accumulator register r of tile t is value(t, r), of row row0 +
// 4 half + 8 (r / 4) + r % 4, half being the lane's half of the wave and row0 the wave's.  V > 1 only where rows are a whole number of V, so that all or none of a lane's
// columns exist.  Every lane of the wave has to call it.
// A lane's place within a group of rows is 32 bits for each array, and the rest of an address the wave's (scalar): addresses of 64 bits a lane and row take what
// registers the accumulators leave.
template <typename T, int V, typename F>
__device__ __forceinline__ void rp_then(const RowProductArgs& g, int64_t row0, int half, int col, F&& value)
{
    constexpr int kBatch = V == 4 ? 4 : 8;
    constexpr int kLanes = 32 / V;          // that share a word of the mask
    const RowProductEpilogue& e = g.then;
    const int64_t rows = g.m - row0 - 4 * half;
    const int left = col < g.n ? (rows < 64 ? (int)rows : 64) : 0;  // rows of the lane, from its first
    auto place = [&](int64_t ld) { return (uint32_t)(4 * half * (int)ld + col) * (uint32_t)sizeof(T); };
    const uint32_t at_c = place(g.ldc), at_r = place(e.ldr), at_z = place(e.ldz);
    uint32_t words[V == 4 ? 2 : 1];  // of the mask, of row number lane % kLanes (and that plus kLanes): all lanes store at once what one of each kLanes would row by row
    auto row_of = [&](const void* base, int64_t ld, int r) { return static_cast<const char*>(base) + (row0 + 8 * (r / 4) + r % 4) * ld * (int64_t)sizeof(T); };
    // Residuals are on their way many rows at a time: a few at a time, 87 K x 512 x 256 in bf16 took 95 us where none took 50.
    constexpr int kAhead = RpHeld<T, V>::kWords > 2 ? 8 : 16;
    RpHeld<T, V> held[kAhead];
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += kBatch) {
        if (r0 % kAhead == 0 && e.residual != nullptr) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int r = r0 + i;
                if (8 * (r / 4) + r % 4 < left) held[i].load(reinterpret_cast<const T*>(row_of(e.residual, e.ldr, r) + at_r));
            }
        }
        float v[kBatch][V];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int t = 0; t < V; ++t) v[i][t] = value(t, r0 + i);
        if (e.z != nullptr) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int r = r0 + i;
                if (8 * (r / 4) + r % 4 < left) rp_store<T, V>(reinterpret_cast<T*>(const_cast<char*>(row_of(e.z, e.ldz, r)) + at_z), v[i]);
            }
        }
        if (e.mask != nullptr) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int r = r0 + i;
                uint32_t word;
                if constexpr (V == 1) {
                    const unsigned long long b = __ballot(left > 0 && act_passes(v[i][0]));
                    word = half == 0 ? (uint32_t)b : (uint32_t)(b >> 32);
                } else {
                    uint32_t bits = 0;
#pragma unroll
                    for (int t = 0; t < V; ++t) bits |= left > 0 && act_passes(v[i][t]) ? 1u << t : 0u;
                    word = group_or<kLanes>(bits << (V * (lane_id() % kLanes)));
                }
                if (lane_id() % kLanes == r % kLanes) words[r / kLanes] = word;
            }
        }
        act_apply<kBatch, V>(e.act, v);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i;
            if (e.residual != nullptr) {
#pragma unroll
                for (int t = 0; t < V; ++t) v[i][t] += held[r % kAhead].at(t);
            }
            if (8 * (r / 4) + r % 4 < left) rp_store<T, V>(reinterpret_cast<T*>(const_cast<char*>(row_of(g.c, g.ldc, r)) + at_c), v[i]);
        }
    }
    if (e.mask != nullptr && (V != 1 || lane_id() % kLanes < 16)) {
#pragma unroll
        for (int q = 0; q < (V == 4 ? 2 : 1); ++q) {
            const int r = q * kLanes + lane_id() % kLanes, row = 8 * (r / 4) + r % 4;
            // (a lane whose columns do not exist stores a row's word all the same, if the word does)
            if (row < rows && col - V * (lane_id() % kLanes) < g.n) (e.mask + row0 * e.mask_ld)[(4 * half + row) * (int)e.mask_ld + col / 32] = words[q];
        }
    }
}

// fp32 products on the bf16 matrix cores: whether they pay for these sizes, and one of them
bool split_product_pays(const RowProductArgs& g);
int split_product(const RowProductArgs& g, bool b_transposed, int form, hipStream_t stream);

// Row blocks, eight at a time, of a kernel that keeps B's columns on the CUs (fgl_split_product.hip)
int64_t sp_row_blocks(int64_t row_tiles, int waves, int per_cu, int64_t tiles_n);

// bf16 products with B kept on the CUs, side[0]'s with bias and epilogue: whether they pay for these sizes, and one of them
bool bf16_product_pays(const RowProductArgs& g);
int bf16_product(const RowProductArgs& g, bool b_transposed, hipStream_t stream);

// side[0]'s product, B transposed or (without an epilogue) not, and its epilogue; sizes, strides and pointers have been checked (bf16: rows of A and B start on words)
int row_product_then(const RowProductArgs& g, bool b_transposed, int dtype, hipStream_t stream);

}  // namespace fgl
