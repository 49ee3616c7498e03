// What the kernels of a dense layer's product over rows share: operands, and how a lane's columns of a row are stored.
#pragma once

#include "fgl_activation.hpp"
#include "fgl_common.hpp"

#include <type_traits>

namespace fgl {

struct RowProductSide {
    const void* a;
    const void* b;
    int64_t lda, ldb;
    int k;  // 0: no such pair
};
// What follows a product: C = act(A B + bias) + residual, and act's derivative, a value or a bit for each
struct RowProductEpilogue {
    int act;               // kActNone ..
    const void* residual;  // (may be null) of C's sizes
    int64_t ldr;
    void* slope;           // (may be null) gelu, silu: the derivative, fp32 or, where C is bf16, fp16 times kSlopeScale
    int64_t lds;
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

// V values as words of memory: fp32, bf16, or (KIND 1) derivatives beside bf16, fp16 times kSlopeScale
template <typename T, int V, int KIND>
struct RpWords {
    static constexpr int kWords = sizeof(T) == 4 ? V : (V + 1) / 2;
    static __device__ __forceinline__ void pack(const float (&v)[V], uint32_t (&w)[kWords])
    {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int t = 0; t < V; ++t) w[t] = __float_as_uint(v[t]);
        } else {
            using E = std::conditional_t<KIND == 1, _Float16, __bf16>;
            typedef E E2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int t = 0; t < V; t += 2) {
                E2 h;
                const float scale = KIND == 1 ? kSlopeScale : 1.0f;
                h[0] = (E)(v[t] * scale);
                h[1] = (E)(v[t + 1 < V ? t + 1 : t] * scale);
                w[t / 2] = __builtin_bit_cast(uint32_t, h);
            }
        }
    }
    static __device__ __forceinline__ void store(char* p, const uint32_t (&w)[kWords])
    {
        if constexpr (sizeof(T) == 2 && V == 1) {
            *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
        } else {
            typedef uint32_t Vec __attribute__((ext_vector_type(kWords), aligned(4)));
            Vec o;
#pragma unroll
            for (int k = 0; k < kWords; ++k) o[k] = w[k];
            *reinterpret_cast<Vec*>(p) = o;
        }
    }
};

// Rows r0 and those after it to memory.  Where `pairs` (rows are a whole number of 2 V columns), neighbouring lanes exchange halves of two rows and each stores 2 V columns of one of
// them: half of the instructions.  (bf16, V = 2, 2.4 M x 100 x 64: with silu and its slopes 300 us in words, 284 in pairs; 87 K x 512 x 256 with a residual 63, 57.)
// row_of(r): where row r of the lane's 16 begins (the wave's), at: the lane's place from there, left: rows of the lane
template <typename T, int V, int KIND, int N, typename F>
__device__ __forceinline__ void rp_store_rows(int r0, const float (&v)[N][V], bool pairs, uint32_t at, int64_t ld, int left, F&& row_of)
{
    using W = RpWords<T, V, KIND>;
    constexpr int NW = W::kWords;
    constexpr bool kPairs = V > 1 && NW <= 2;
    const uint32_t odd = (uint32_t)lane_id() & 1u;
    const uint32_t at_pair = at + (odd != 0 ? (uint32_t)ld * (uint32_t)sizeof(T) - 4u * NW : 0u);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const int r = r0 + i, row = 8 * (r / 4) + r % 4;
        uint32_t a[NW], b[NW];
        W::pack(v[i], a);
        W::pack(v[i + 1], b);
        if (kPairs && pairs) {
            typedef uint32_t Vec __attribute__((ext_vector_type(2 * NW), aligned(4)));
            Vec o;
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const uint32_t got = dpp_u32<kDppXor1>(odd != 0 ? a[k] : b[k]);
                o[k] = odd != 0 ? got : a[k];
                o[NW + k] = odd != 0 ? b[k] : got;
            }
            if (row + (int)odd < left) *reinterpret_cast<Vec*>(row_of(r) + at_pair) = o;
        } else {
            if (row < left) W::store(row_of(r) + at, a);
            if (row + 1 < left) W::store(row_of(r + 1) + at, b);
        }
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
    constexpr int kBatch = 4;
    constexpr int kLanes = 32 / V;          // that share a word of the mask
    const RowProductEpilogue& e = g.then;
    const int64_t rows = g.m - row0 - 4 * half;
    const int left = col < g.n ? (rows < 64 ? (int)rows : 64) : 0;  // rows of the lane, from its first
    auto place = [&](int64_t ld) { return (uint32_t)(4 * half * (int)ld + col) * (uint32_t)sizeof(T); };
    const uint32_t at_c = place(g.ldc), at_r = place(e.ldr), at_s = place(e.lds);
    uint32_t words[V == 4 ? 2 : 1];  // of the mask, of row number lane % kLanes (and that plus kLanes): all lanes store at once what one of each kLanes would row by row
    auto row_of = [&](const void* base, int64_t ld, int r) { return static_cast<char*>(const_cast<void*>(base)) + (row0 + 8 * (r / 4) + r % 4) * ld * (int64_t)sizeof(T); };
    const bool pairs = g.n % (2 * V) == 0;
    // Residuals are on their way many rows at a time: a few at a time, 87 K x 512 x 256 in bf16 took 95 us where none took 50.
    constexpr int kAhead = RpHeld<T, V>::kWords > 2 ? 4 : 8;
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
        if (e.slope != nullptr) {
            float slope[kBatch][V];
            act_with_slope<kBatch, V>(e.act, v, slope);
            rp_store_rows<T, V, 1>(r0, slope, pairs, at_s, e.lds, left, [&](int r) { return row_of(e.slope, e.lds, r); });
        } else {
            act_apply<kBatch, V>(e.act, v);
        }
        if (e.residual != nullptr) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
                for (int t = 0; t < V; ++t) v[i][t] += held[(r0 + i) % kAhead].at(t);
        }
        rp_store_rows<T, V, 0>(r0, v, pairs, at_c, g.ldc, left, [&](int r) { return row_of(g.c, g.ldc, r); });
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
