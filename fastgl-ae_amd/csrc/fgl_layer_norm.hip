// Norm of the rows of a matrix and its gradients:
//   h = (x - mean) / sqrt(var + eps),   y = h w + b,   relu: y = max(y, 0)
//   g = dy [y > 0] w,   dx = (g - mean(g) - h mean(g h)) / sqrt(var + eps),   dw = sum over rows of dy [y > 0] h,   db = sum of dy [y > 0]
//
// One pass over the rows each way: 4 (fp32: 8), 16 or 64 lanes hold a row in registers, 16 bytes a lane and load, so a wave has 16 (8), 4 or one of them; sums
// over a row are exchanges between its lanes.  In the backward pass a lane adds up dw and db of its columns over all rows that its wave takes, a
// workgroup those of its waves through LDS, and a second launch those of the workgroups, in a fixed order.
//
// Mean, variance and h are formed in 64 bits: rows far from zero keep what they differ in (a mean in 32 bits is off by 2^-24 of itself, which may be more
// than the row's spread), relu's decision and the code of a value in 8 bits (fgl_keep8.hpp) are those of the formula, not of an order of summation.
// The 64-bit instructions issue like the 32-bit ones here, and there is room for them beside the pass over memory; but where a bf16 row's codes and relu's decision are formed too, they
// are what the forward pass takes.
//
// For the backward pass a row leaves its mean (64 bits) and 1 / sqrt (32, of a wider range: it, and differences from the mean, may be past fp32's where h is not), with relu a bit a value, and with KEEP8 h in 8 bits a value in x's place.
//
// What bounds it: the pass over memory.  us forward / back (and 4 .. 7 for the second launch): 60 K x 256 fp32 22 / 37 (5.6 and 4.9 TB/s; relu in it), 87 K x 256 bf16 with relu and KEEP8
// 27 / 28, where the 64-bit instructions of codes and relu's decision take longer than the memory forward, 2.4 M x 64 fp32 of rows of 100 columns with KEEP8 325 / 266.  Rows that do not begin on 16 bytes cost
// loads and stores across lines: 200 K x 602 bf16 137 / 191, 600 columns 107 / 161.
#include "fgl_common.hpp"
#include "fgl_keep8.hpp"
#include "fgl_kernels.hpp"

#include <type_traits>

namespace fgl {

constexpr int kLnThreads = 512, kLnWaves = kLnThreads / kWave;
constexpr int kLnMostCols = 2048;
constexpr int kLnMostBlocks = 1024;  // of the backward pass: rows of partial sums

struct LnState {
    double* mean;    // without KEEP8
    float* rstd;     // ln_held
    uint8_t* mask;   // relu: [n][mask_ld], bit c % 8 of byte c / 8
    uint8_t* codes;  // KEEP8: [n][k8_columns(d)]
    uint8_t* steps;  // KEEP8: [n][k8_columns(d) / 32]
    size_t bytes;
};

static LnState ln_state(void* base, int64_t n, int d, bool relu, bool keep8)
{
    Carver c(base);
    LnState s;
    memset(&s, 0, sizeof(s));
    if (!keep8) s.mean = c.take<double>((size_t)n);
    s.rstd = c.take<float>((size_t)n);
    if (relu) s.mask = c.take<uint8_t>((size_t)n * (size_t)((d + 7) / 8));
    if (keep8) {
        s.codes = c.take<uint8_t>((size_t)n * (size_t)k8_columns(d));
        s.steps = c.take<uint8_t>((size_t)n * (size_t)(k8_columns(d) / 32));
    }
    s.bytes = c.used();
    return s;
}

struct LnArgs {
    const void* x;
    const void* dy;
    const void* w;  // (may be null: ones)
    const void* b;  // (may be null: zeros)
    void* y;
    void* dx;       // (may be null)
    float* partial; // [workgroup][2][d]: dw, db (null: neither is wanted)
    LnState state;  // (forward: rstd null where nothing is kept)
    int64_t n, ldx, lddy;
    int d, mask_ld, code_ld;
    int relu;
    double eps;
    float inv_d;
    double inv_d64;
};

template <typename T>
constexpr int kLnV = 16 / (int)sizeof(T);
template <typename T>
using LnVec = T __attribute__((ext_vector_type(kLnV<T>), aligned(sizeof(T))));

// sums over the G lanes of a row, the same in all of them
template <int G>
__device__ __forceinline__ double ln_sum(double v)
{
    auto add = [&](auto ctrl) {
        const uint32_t lo = dpp_u32<decltype(ctrl)::value>((uint32_t)__double2loint(v)), hi = dpp_u32<decltype(ctrl)::value>((uint32_t)__double2hiint(v));
        v += __hiloint2double((int)hi, (int)lo);
    };
    add(std::integral_constant<int, kDppXor1>{});
    add(std::integral_constant<int, kDppXor2>{});
    if constexpr (G >= 8) add(std::integral_constant<int, kDppHalfMirror>{});
    if constexpr (G >= 16) add(std::integral_constant<int, kDppMirror>{});
    if constexpr (G == 64) {
        v += __shfl_xor(v, 16, kWave);
        v += __shfl_xor(v, 32, kWave);
    }
    return v;
}
template <int G>
__device__ __forceinline__ float ln_sum(float v)
{
    v += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(v)));
    v += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(v)));
    if constexpr (G >= 8) v += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(v)));
    if constexpr (G >= 16) v += __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(v)));
    if constexpr (G == 64) {
        v += __shfl_xor(v, 16, kWave);
        v += __shfl_xor(v, 32, kWave);
    }
    return v;
}

// 1 / sqrt(v) from the instruction's 2^-25 or so: with e = 1 - v r^2, r (1 - e)^-1/2 = r (1 + e / 2 + 3 e^2 / 8 + ..)
__device__ __forceinline__ double ln_rsqrt(double v)
{
    const double r = __builtin_amdgcn_rsq(v), e = fma(-v * r, r, 1.0);
    return fma(r * e, fma(0.375, e, 0.5), r);
}

// 1 / sqrt in 32 bits: as it is from 2^-100 to 2^100; negative, times 2^-36 above (up to 2^162: rows of one value and an eps below 2^-324 alone have more) and times 2^150 below
__device__ __forceinline__ float ln_held(double r)
{
    if (r > 0x1p100) return -(float)(fmin(r, 0x1p162) * 0x1p-36);
    if (r < 0x1p-100) return -(float)(r * 0x1p150);
    return (float)r;
}
__device__ __forceinline__ double ln_of_held(float v)
{
    const double r = v;
    return v < 0.0f ? r * (v < -0x1p57f ? -0x1p36 : -0x1p-150) : r;
}

// The lane's values of a chunk, of which the first `left` exist (others: `fill`).  WHOLE: rows are a whole number of chunks, all or none exist.
template <bool WHOLE, typename T>
__device__ __forceinline__ LnVec<T> ln_load(const T* p, bool inside, int left, float fill = 0.0f)
{
    LnVec<T> v;
    if (inside || left >= kLnV<T>) {
        v = *reinterpret_cast<const LnVec<T>*>(p);
    } else {
#pragma unroll
        for (int e = 0; e < kLnV<T>; ++e) v[e] = (T)fill;
        if constexpr (!WHOLE) {
#pragma unroll
            for (int e = 0; e < kLnV<T>; ++e)
                if (e < left) v[e] = p[e];
        }
    }
    return v;
}
// Of a lane's loads, how many lie within the row whatever the row (ln_shape): those that a shape with fewer would have
constexpr int ln_inside(int lanes, int loads) { return lanes < 16 ? 0 : loads == 8 ? 6 : lanes == 64 && loads == 6 ? 4 : loads - 1; }
template <bool WHOLE>
__device__ __forceinline__ bool ln_there(bool inside, int e, int left) { return inside || (WHOLE ? left > 0 : e < left); }
// Keeps what is made of a parameter (its 32 or 64-bit value) from being formed before the loop over rows and held in twice or four times the registers
template <typename T>
__device__ __forceinline__ void ln_as_held(LnVec<T>& v)
{
    typedef uint32_t U4 __attribute__((ext_vector_type(4)));
    U4 u = __builtin_bit_cast(U4, v);
    asm volatile("" : "+v"(u));
    v = __builtin_bit_cast(LnVec<T>, u);
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void ln_store(T* p, bool inside, int left, const LnVec<T>& v)
{
    if (inside || left >= kLnV<T>) {
        *reinterpret_cast<LnVec<T>*>(p) = v;
    } else if constexpr (!WHOLE) {
#pragma unroll
        for (int e = 0; e < kLnV<T>; ++e)
            if (e < left) p[e] = v[e];
    }
}

// V bytes of codes
template <int V>
using LnCodes = uint32_t __attribute__((ext_vector_type(V / 4)));

template <typename T, int G, int C, bool KEEP8, bool WHOLE>
__global__ __launch_bounds__(kLnThreads, C * kLnV<T> <= 16 ? 4 : 2) void layer_norm_kernel(const LnArgs g)
{
    constexpr int V = kLnV<T>, kRows = kWave / G;
    constexpr int kGroup = 32 / V;  // lanes that share a step
    const int lane = lane_id(), l = lane % G;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const T* x = static_cast<const T*>(g.x);
    T* y = static_cast<T*>(g.y);
    LnVec<T> w[C], b[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int c = (j * G + l) * V, left = g.d - c;
        w[j] = ln_load<WHOLE>(static_cast<const T*>(g.w) + c, false, g.w != nullptr ? left : 0, 1.0f);
        b[j] = ln_load<WHOLE>(static_cast<const T*>(g.b) + c, false, g.b != nullptr ? left : 0, 0.0f);
    }
    const int64_t stride = (int64_t)gridDim.x * kLnWaves * kRows;
    for (int64_t row0 = ((int64_t)blockIdx.x * kLnWaves + wave) * kRows; row0 < g.n; row0 += stride) {
        const bool mine = row0 + lane / G < g.n;
        const int64_t row = mine ? row0 + lane / G : g.n - 1;  // (past the end: the last row again, not stored)
        LnVec<T> v[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            ln_as_held<T>(w[j]);
            ln_as_held<T>(b[j]);
            const int c = (j * G + l) * V;
            v[j] = ln_load<WHOLE>(x + row * g.ldx + c, j < ln_inside(G, C), g.d - c);
        }
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) sum += (double)(float)v[j][e];
        sum = ln_sum<G>(sum);
        double mean = sum * g.inv_d64;
        mean = fma(fma(-mean, (double)g.d, sum), g.inv_d64, mean);  // (the quotient itself: a row of one value has no spread)
        double square = 0.0;
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double t = (double)(float)v[j][e] - mean;
                if (ln_there<WHOLE>(j < ln_inside(G, C), e, g.d - (j * G + l) * V)) square = fma(t, t, square);
            }
        const double rstd = ln_rsqrt(fma(ln_sum<G>(square), g.inv_d64, g.eps));
        if (g.state.rstd != nullptr && l == 0 && mine) {
            g.state.rstd[row] = ln_held(rstd);
            if constexpr (!KEEP8) g.state.mean[row] = mean;
        }
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int c = (j * G + l) * V, left = g.d - c;
            double h[V];
            float out[V];
#pragma unroll
            for (int e = 0; e < V; ++e) h[e] = ln_there<WHOLE>(j < ln_inside(G, C), e, left) ? ((double)(float)v[j][e] - mean) * rstd : 0.0;
            if (g.relu) {
                uint32_t bits = 0;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const double t = fma(h[e], (double)(float)w[j][e], (double)(float)b[j][e]);
                    bits |= t <= 0.0 ? 0u : 1u << e;
                    out[e] = t <= 0.0 ? 0.0f : (float)t;  // (what is not a number stays it)
                }
                if (V == 4) bits |= dpp_u32<kDppXor1>(bits) << 4;  // (the even lane's)
                if (g.state.mask != nullptr && mine && left > 0 && (V == 8 || l % 2 == 0)) g.state.mask[row * g.mask_ld + c / 8] = (uint8_t)bits;
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) out[e] = fmaf((float)h[e], (float)w[j][e], (float)b[j][e]);
            }
            LnVec<T> q;
#pragma unroll
            for (int e = 0; e < V; ++e) q[e] = (T)out[e];
            if (mine) ln_store<WHOLE>(y + row * g.d + c, j < ln_inside(G, C), left, q);
            if constexpr (KEEP8) {
                uint32_t most = 0;  // the largest magnitude's upper word: exponent and first bits
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const uint32_t m = (uint32_t)__double2hiint(h[e]) & 0x7FFFFFFFu;
                    most = most > m ? most : m;
                }
                most = group_max<kGroup>(most) >> 20;
                const uint32_t step = most == 0x7FF ? kStepNone : k8_step((int)most - 1023);
                const double inverse = step == kStepNone ? 0.0 : k8_inverse64(step);
                LnCodes<V> codes;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const uint32_t code = k8_code(h[e], inverse);
                    if (e % 4 == 0) codes[e / 4] = code;
                    else codes[e / 4] |= code << 8 * (e % 4);
                }
                codes ^= kSigned;
                if (mine && c < g.code_ld) {
                    *reinterpret_cast<LnCodes<V>*>(g.state.codes + row * g.code_ld + c) = codes;
                    if (l % kGroup == 0) g.state.steps[row * (g.code_ld / 32) + c / 32] = (uint8_t)step;
                }
            }
        }
    }
}

template <typename T, int G, int C, bool KEEP8, bool WHOLE>
__global__ __launch_bounds__(kLnThreads, C * kLnV<T> <= 16 ? 4 : 2) void layer_norm_backward_kernel(const LnArgs g)
{
    constexpr int V = kLnV<T>, kRows = kWave / G;
    __shared__ float s_sum[kLnWaves][2][G * V];
    const int lane = lane_id(), l = lane % G;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const T* x = static_cast<const T*>(g.x);
    const T* dy = static_cast<const T*>(g.dy);
    T* dx = static_cast<T*>(g.dx);
    LnVec<T> w[C];
    float dw[C][V], db[C][V];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int c = (j * G + l) * V;
        w[j] = ln_load<WHOLE>(static_cast<const T*>(g.w) + c, false, g.w != nullptr ? g.d - c : 0, 1.0f);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[j][e] = db[j][e] = 0.0f;
    }
    const int64_t stride = (int64_t)gridDim.x * kLnWaves * kRows;
    for (int64_t row0 = ((int64_t)blockIdx.x * kLnWaves + wave) * kRows; row0 < g.n; row0 += stride) {
        const bool mine = row0 + lane / G < g.n;
        const int64_t row = mine ? row0 + lane / G : g.n - 1;
        float h[C][V], t[C][V];
        LnVec<T> vx[C], vd[C];
        LnCodes<V> codes[C];
        uint32_t step[C], bits[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            ln_as_held<T>(w[j]);
            const int c = (j * G + l) * V, left = g.d - c;
            vd[j] = ln_load<WHOLE>(dy + row * g.lddy + c, false, mine ? left : 0);  // (past the end: zeros, which add nothing)
            if constexpr (KEEP8) {
                const int at = c < g.code_ld ? c : 0;
                codes[j] = *reinterpret_cast<const LnCodes<V>*>(g.state.codes + row * g.code_ld + at);
                step[j] = g.state.steps[row * (g.code_ld / 32) + at / 32];
            } else {
                vx[j] = ln_load<WHOLE>(x + row * g.ldx + c, j < ln_inside(G, C), left);
            }
            bits[j] = 0xFFu;
            if (g.relu && left > 0) bits[j] = (uint32_t)g.state.mask[row * g.mask_ld + c / 8] >> (c % 8);
        }
        const double rstd = ln_of_held(g.state.rstd[row]);
        const double mean = KEEP8 ? 0.0 : g.state.mean[row];
        float sum = 0.0f, with_h = 0.0f;
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const bool there = ln_there<WHOLE>(j < ln_inside(G, C), e, g.d - (j * G + l) * V);
                if constexpr (KEEP8) h[j][e] = there ? k8_code_value(codes[j][e / 4], e % 4) * k8_step_value(step[j]) : 0.0f;
                else h[j][e] = there ? (float)(((double)(float)vx[j][e] - mean) * rstd) : 0.0f;
                const float d = bits[j] >> e & 1u ? (float)vd[j][e] : 0.0f;
                // (rows past the end leave dw as it is, also where the last one's h is no number)
                dw[j][e] = fmaf(d, mine ? h[j][e] : 0.0f, dw[j][e]);
                db[j][e] += d;
                t[j][e] = d * (float)w[j][e];
                sum += t[j][e];
                with_h = fmaf(t[j][e], h[j][e], with_h);
            }
        if (dx == nullptr) continue;
        sum = ln_sum<G>(sum) * g.inv_d;
        with_h = ln_sum<G>(with_h) * g.inv_d;
        // bf16: 1 / sqrt in two factors, the second a power of two, one unless the whole is next to fp32's ends or past them (rows of tiny values without eps, rows next to the
        // largest).  fp32: in 64 bits, which cost less there than the registers of the factors, and more than they in bf16 (us forward and back: 60 K x 256 fp32 64.3 / 66.4 in factors,
        // 200 K x 602 bf16 335 / 330).
        const float more = rstd > 0x1p100 ? 0x1p100f : rstd < 0x1p-100 ? 0x1p-100f : 1.0f;
        const float scale = (float)(rstd * (rstd > 0x1p100 ? 0x1p-100 : rstd < 0x1p-100 ? 0x1p100 : 1.0));
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int c = (j * G + l) * V;
            LnVec<T> q;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float v = t[j][e] - sum - h[j][e] * with_h;
                if constexpr (sizeof(T) == 4) q[e] = (float)(rstd * (double)v);
                else q[e] = (T)(scale * v * more);
            }
            if (mine) ln_store<WHOLE>(dx + row * g.d + c, j < ln_inside(G, C), g.d - c, q);
        }
    }
    if (g.partial == nullptr) return;
    float* out = g.partial + (int64_t)blockIdx.x * 2 * g.d;
#pragma unroll
    for (int j = 0; j < C; ++j) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float a = dw[j][e], b = db[j][e];
#pragma unroll
            for (int s = G; s < kWave; s *= 2) {
                a += __shfl_xor(a, s, kWave);
                b += __shfl_xor(b, s, kWave);
            }
            if (lane < G) {
                s_sum[wave][0][lane * V + e] = a;
                s_sum[wave][1][lane * V + e] = b;
            }
        }
        __syncthreads();
        for (int i = (int)threadIdx.x; i < 2 * G * V; i += kLnThreads) {
            const int which = i / (G * V), c = i % (G * V);
            float s = s_sum[0][which][c];
#pragma unroll
            for (int k = 1; k < kLnWaves; ++k) s += s_sum[k][which][c];
            if (j * G * V + c < g.d) out[which * g.d + j * G * V + c] = s;
        }
        __syncthreads();
    }
}

// dw and db from the workgroups' sums: 32 columns a workgroup, 32 lanes of rows, eight loads of each on their way (of 1024 rows of 2 x 256 columns: 12 us with
// a quarter of the lanes and half of the loads, 4 so)
constexpr int kLnReduce = 1024;
template <typename T>
__global__ __launch_bounds__(kLnReduce) void layer_norm_reduce_kernel(const float* __restrict__ partial, int rows, int d, T* __restrict__ dw, T* __restrict__ db)
{
    constexpr int kLanes = kLnReduce / 32, kBatch = 8;
    __shared__ float s_sum[kLanes][33];
    const int i = (int)(threadIdx.x % 32), r = (int)(threadIdx.x / 32), c = (int)blockIdx.x * 32 + i;
    float s = 0.0f;
    if (c < 2 * d) {
        for (int q = r; q < rows; q += kLanes * kBatch) {
            float v[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) v[k] = q + k * kLanes < rows ? partial[(int64_t)(q + k * kLanes) * 2 * d + c] : 0.0f;
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
    }
    s_sum[r][i] = s;
    __syncthreads();
    if (r != 0 || c >= 2 * d) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < kLanes; k += 4) s += (s_sum[k][i] + s_sum[k + 1][i]) + (s_sum[k + 2][i] + s_sum[k + 3][i]);
    if (c < d) {
        if (dw != nullptr) dw[c] = (T)s;
    } else if (db != nullptr) {
        db[c - d] = (T)s;
    }
}

// Lanes of a row and loads of a lane.  16 lanes as long as their registers hold a row: four rows a wave share what is done once a row, sums over 16 lanes need no
// exchange through LDS, and a lane has many loads on their way (200 K x 602 in bf16, of
// which 64 lanes would take two loads each and leave two fifths of them empty: 235 us forward and 265 back, 137 and 191 so).
// In bf16 a row of more than 48 elements a lane takes 64 lanes,
// in the backward pass, where a lane holds four values for each, two of them sums, one of more than 40.
struct LnShape {
    int lanes, loads;
};
static LnShape ln_shape(int d, int v, bool backward)
{
    const int chunks = (d + v - 1) / v;
    if (chunks <= 32 / v) return {32 / v, 1};
    const int most = v == 4 ? 128 : backward ? 80 : 96;
    if (chunks <= most) return {16, chunks > 96 ? 8 : (chunks + 15) / 16};
    const int loads = (chunks + 63) / 64;
    return {64, loads > 6 ? 8 : loads > 4 ? 6 : loads};
}

// Calls f with integral constants: ln_shape's lanes and loads, whether rows are whole numbers of loads.
template <typename T, bool BACKWARD, typename F>
static void ln_dispatch(int d, F&& f)
{
    constexpr int V = kLnV<T>;
    const LnShape s = ln_shape(d, V, BACKWARD);
    auto call = [&](auto lanes, auto loads) {
        if (s.lanes != decltype(lanes)::value || s.loads != decltype(loads)::value) return;
        if (d % V == 0) f(lanes, loads, std::true_type{});
        else f(lanes, loads, std::false_type{});
    };
    auto each = [&](auto lanes, auto... loads) { (call(lanes, loads), ...); };
    using std::integral_constant;
    constexpr integral_constant<int, 1> k1{};
    constexpr integral_constant<int, 2> k2{};
    constexpr integral_constant<int, 3> k3{};
    constexpr integral_constant<int, 4> k4{};
    constexpr integral_constant<int, 5> k5{};
    constexpr integral_constant<int, 6> k6{};
    constexpr integral_constant<int, 8> k8{};
    constexpr integral_constant<int, 16> k16{};
    constexpr integral_constant<int, 64> k64{};
    call(integral_constant<int, 32 / V>{}, k1);
    each(k16, k1, k2, k3, k4, k5);
    if constexpr (V == 4 || !BACKWARD) call(k16, k6);
    if constexpr (V == 4) call(k16, k8);
    else call(k64, k2);
    each(k64, k3, k4);
    if constexpr (V == 4) each(k64, k6, k8);
}

static int64_t ln_blocks(int64_t n, int d, int dtype, bool backward, int64_t most)
{
    const int rows = kWave / ln_shape(d, dtype == FGL_F32 ? 4 : 8, backward).lanes * kLnWaves;
    const int64_t want = ceil_div(n, rows);
    return want < most ? want : most;
}

static bool ln_sizes(int64_t n, int d, int dtype) { return n >= 0 && n <= (1LL << 31) && d >= 1 && d <= kLnMostCols && (dtype == FGL_F32 || dtype == FGL_BF16); }

static LnArgs ln_args(int64_t n, int d, double eps, int relu)
{
    LnArgs g;
    memset(&g, 0, sizeof(g));
    g.n = n;
    g.d = d;
    g.mask_ld = (d + 7) / 8;
    g.code_ld = (int)k8_columns(d);
    g.relu = relu != 0;
    g.eps = eps;
    g.inv_d64 = 1.0 / d;
    g.inv_d = (float)g.inv_d64;
    return g;
}

}  // namespace fgl

using namespace fgl;

FGL_EXPORT size_t fgl_layer_norm_state_bytes(int64_t n, int d, int relu, int keep8)
{
    return ln_sizes(n, d, FGL_F32) ? ln_state(nullptr, n, d, relu != 0, keep8 != 0).bytes : 0;
}

FGL_EXPORT size_t fgl_layer_norm_workspace_bytes(int64_t n, int d, int dtype)
{
    return ln_sizes(n, d, dtype) ? (size_t)ln_blocks(n, d, dtype, true, kLnMostBlocks) * 2 * (size_t)d * sizeof(float) : 0;
}

FGL_EXPORT int fgl_layer_norm(const void* d_x, int64_t ldx, const void* d_w, const void* d_b, int64_t n, int d, int dtype, double eps, int relu, int keep8,
                              void* d_y, void* d_state, size_t state_bytes, void* stream)
{
    FGL_REQUIRE(ln_sizes(n, d, dtype), "layer_norm: %lld rows of %d columns, dtype %d", (long long)n, d, dtype);
    FGL_REQUIRE(ldx >= d, "layer_norm: row stride smaller than the row length");
    FGL_REQUIRE(eps >= 0.0 && eps < 1e300, "layer_norm: eps %g", eps);
    if (n == 0) return FGL_OK;
    FGL_REQUIRE(d_x && d_y, "layer_norm: null pointer");
    LnArgs g = ln_args(n, d, eps, relu);
    g.x = d_x; g.ldx = ldx; g.w = d_w; g.b = d_b; g.y = d_y;
    if (d_state != nullptr) {
        g.state = ln_state(d_state, n, d, relu != 0, keep8 != 0);
        if (state_bytes < g.state.bytes || ((uintptr_t)d_state & 255) != 0) {
            set_error("layer_norm: state of %zu bytes at a multiple of 256 bytes, %zu given", g.state.bytes, state_bytes);
            return FGL_ERR_WORKSPACE;
        }
    }
    const bool codes = keep8 != 0 && d_state != nullptr;
    const dim3 grid((unsigned)ln_blocks(n, d, dtype, false, 4096));
    auto launch = [&](auto type) {
        using T = decltype(type);
        ln_dispatch<T, false>(d, [&](auto lanes, auto loads, auto whole) {
            constexpr int G = decltype(lanes)::value, C = decltype(loads)::value;
            constexpr bool W = decltype(whole)::value;
            if (codes) hipLaunchKernelGGL((layer_norm_kernel<T, G, C, true, W>), grid, dim3(kLnThreads), 0, as_stream(stream), g);
            else hipLaunchKernelGGL((layer_norm_kernel<T, G, C, false, W>), grid, dim3(kLnThreads), 0, as_stream(stream), g);
        });
    };
    if (dtype == FGL_F32) launch(float{});
    else launch(__bf16{});
    FGL_CHECK_LAUNCH("layer_norm_kernel");
    return FGL_OK;
}

FGL_EXPORT int fgl_layer_norm_backward(const void* d_dy, int64_t lddy, const void* d_x, int64_t ldx, const void* d_w, int64_t n, int d, int dtype, int relu,
                                       int keep8, const void* d_state, size_t state_bytes, void* d_dx, void* d_dw, void* d_db, void* d_ws, size_t ws_bytes,
                                       void* stream)
{
    FGL_REQUIRE(ln_sizes(n, d, dtype) && n >= 1, "layer_norm_backward: %lld rows of %d columns, dtype %d", (long long)n, d, dtype);
    FGL_REQUIRE(lddy >= d && (keep8 || ldx >= d), "layer_norm_backward: row stride smaller than the row length");
    FGL_REQUIRE(d_dy && d_state && (keep8 || d_x), "layer_norm_backward: null pointer");
    LnArgs g = ln_args(n, d, 0.0, relu);
    g.state = ln_state(const_cast<void*>(d_state), n, d, relu != 0, keep8 != 0);
    if (state_bytes < g.state.bytes || ((uintptr_t)d_state & 255) != 0) {
        set_error("layer_norm_backward: state of %zu bytes at a multiple of 256 bytes, %zu given", g.state.bytes, state_bytes);
        return FGL_ERR_WORKSPACE;
    }
    const bool sums = d_dw != nullptr || d_db != nullptr;
    if (d_dx == nullptr && !sums) return FGL_OK;
    const int64_t blocks = ln_blocks(n, d, dtype, true, kLnMostBlocks);
    if (sums && (d_ws == nullptr || ws_bytes < (size_t)blocks * 2 * d * sizeof(float) || ((uintptr_t)d_ws & 255) != 0)) {
        set_error("layer_norm_backward: workspace too small (%zu < %zu) or not at a multiple of 256 bytes", ws_bytes, (size_t)blocks * 2 * d * sizeof(float));
        return FGL_ERR_WORKSPACE;
    }
    g.dy = d_dy; g.lddy = lddy; g.x = d_x; g.ldx = ldx; g.w = d_w; g.dx = d_dx;
    g.partial = sums ? static_cast<float*>(d_ws) : nullptr;
    auto launch = [&](auto type) {
        using T = decltype(type);
        ln_dispatch<T, true>(d, [&](auto lanes, auto loads, auto whole) {
            constexpr int G = decltype(lanes)::value, C = decltype(loads)::value;
            constexpr bool W = decltype(whole)::value;
            if (keep8) hipLaunchKernelGGL((layer_norm_backward_kernel<T, G, C, true, W>), dim3((unsigned)blocks), dim3(kLnThreads), 0, as_stream(stream), g);
            else hipLaunchKernelGGL((layer_norm_backward_kernel<T, G, C, false, W>), dim3((unsigned)blocks), dim3(kLnThreads), 0, as_stream(stream), g);
        });
        if (sums)
            hipLaunchKernelGGL((layer_norm_reduce_kernel<T>), dim3((unsigned)ceil_div(2 * d, 32)), dim3(kLnReduce), 0, as_stream(stream), g.partial, (int)blocks, d,
                               static_cast<T*>(d_dw), static_cast<T*>(d_db));
    };
    if (dtype == FGL_F32) launch(float{});
    else launch(__bf16{});
    FGL_CHECK_LAUNCH("layer_norm_backward_kernel");
    return FGL_OK;
}
